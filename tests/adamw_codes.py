"""What an AdamW step keeps in 8 bits where it rounds at random, by the definition: fp32 numbers to codes and back (any device)."""
import torch

GROUP = 128
WORD = 0xFFFFFFFF


def mix(x):
    x = ((x ^ (x >> 16)) * 0x9E3779B1) & WORD
    x = ((x ^ (x >> 15)) * 0x85A308D3) & WORD
    return x ^ (x >> 16)


def words(index, step):
    """The random words of elements ``index`` (int64) in step ``step``."""
    t = torch.tensor([step & WORD, step >> 32], device=index.device)
    key = mix((mix(t[0]) + t[1] * 0x9E3779B1 + 0x243F6A88) & WORD)
    return mix(((index & WORD) + (index >> 32) * 0x9E3779B1 + key) & WORD)


def hold(x, bits, word):
    """x fp32 [n]: codes uint8 [n], exponents uint8 [groups] and the values that they stand for.  ``bits`` 3: the moment, 4: the root;
    ``word`` None: to the nearest code."""
    n = x.numel()
    pad = -n % GROUP
    x = torch.nn.functional.pad(x.float(), (0, pad)).view(-1, GROUP)
    shift = 23 - bits
    b = x.abs().view(torch.int32).long()

    def rounded(b):
        if word is None:
            return b + (1 << (shift - 1)) - 1 + (b >> shift & 1)
        half = word & 0xFFFF if bits == 3 else word >> 16
        half = torch.nn.functional.pad(half, (0, pad)).view(-1, GROUP)
        return b + (half << (shift - 16)) + (1 << (shift - 17))

    E = torch.clamp(rounded(b).amax(1, keepdim=True) >> 23, max=255)
    # (the scaled number as an fp32 one, which rounds what is below its normal numbers)
    s = (x.abs().double() * torch.exp2((15 - E).double())).float().view(torch.int32).long()
    if bits == 4:
        s = torch.maximum(s, torch.clamp(b, max=1 << shift))
    code = rounded(s) >> shift
    if word is None:                                         # rounded once: below the normal codes in units of the smallest one
        units = x.abs().double() * torch.exp2((141 + bits - E).double())
        near = torch.round(units).long()
        if bits == 4:
            near = torch.where(x > 0, torch.clamp(near, min=1), near)
        code = torch.where(units < 1 << bits, near, code)
    dead = (E == 0) | (E == 255)
    value = (code << shift).int().view(torch.float32).double() * torch.exp2((E - 15).double())
    value = torch.where(E == 0, 0.0, torch.where(E == 255, torch.nan, torch.where(x < 0, -value, value)))
    if bits == 3:
        code = code + 128 * (x.view(torch.int32) < 0)
    code = torch.where(dead, 0, code)
    return code.to(torch.uint8).view(-1)[:n], E.to(torch.uint8).view(-1), value.float().view(-1)[:n]
