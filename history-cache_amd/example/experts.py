"""Node classification with maps per node type, a layer of experts and activations kept in 8 bits.

A random graph whose nodes have one of three types; what a node's features mean depends on its type.  The model projects the
features by one matrix for each type (``expert_linear``), averages the neighbours (``MySageConvHistory``), sends every node
through its router's choice of experts (``ExpertMLP``) and classifies.  Everything that the layers keep for backward at full
width is kept in 8 bits.

    python experts.py                               # 20 000 nodes, 60 steps
    python experts.py --nodes 200000 --experts 16 --dtype bf16 --full-width
"""
import argparse
import contextlib
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import hiscache  # noqa: E402
import hiscache_backend as be  # noqa: E402
from hiscache.synthetic import uniform_graph  # noqa: E402

TYPES = 3


class Net(torch.nn.Module):
    def __init__(self, features, hidden, classes, experts, top_k, dtype):
        super().__init__()
        self.by_type = torch.nn.Parameter(torch.randn(TYPES, hidden, features) / features ** 0.5)
        self.conv = hiscache.MySageConvHistory(hidden, hidden, need_grad=False)
        self.norm = torch.nn.LayerNorm(hidden)
        self.experts = hiscache.ExpertMLP(hidden, 2 * hidden, experts, top_k, dtype=dtype)
        self.out = torch.nn.Linear(hidden, classes)
        self.dtype = dtype

    def forward(self, x, types, ptr, idx, context):
        order = be.expert_order(types, TYPES)
        with context():
            rows = be.expert_linear(be.rows_to_experts(x, order), self.by_type, order.offset)
            h = be.rows_from_experts(rows, order)
            h, _ = self.conv(h, ptr, idx, None, None, 0, h.shape[0])
            h = F.relu(self.norm(h))
        h = h + self.experts(h.to(self.dtype)).float()
        return self.out(h).log_softmax(1)


def make_data(nodes, features, classes, seed, device):
    gen = torch.Generator().manual_seed(seed)
    indptr, indices = uniform_graph(nodes, 8, seed)
    x = torch.randn(nodes, features, generator=gen)
    types = torch.randint(0, TYPES, (nodes,), generator=gen)
    meaning = torch.randn(TYPES, features, classes, generator=gen)
    y = torch.bmm(x.unsqueeze(1), meaning[types]).squeeze(1).argmax(1)
    to = [torch.as_tensor(t).to(device) for t in (x, types, torch.from_numpy(indptr), torch.from_numpy(indices), y)]
    return to


def run(args, say=print):
    """The losses of all steps."""
    device, dtype = "cuda:0", {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[args.dtype]
    torch.manual_seed(args.seed)
    x, types, ptr, idx, y = make_data(args.nodes, args.features, args.classes, args.seed, device)
    net = Net(args.features, args.hidden, args.classes, args.experts, args.top_k, dtype).to(device).train()
    opt = torch.optim.Adam(net.parameters(), lr=args.lr)
    context = contextlib.nullcontext if args.full_width else hiscache.packed_activations
    losses = []
    for step in range(args.steps):
        before = torch.cuda.memory_allocated()
        loss = F.nll_loss(net(x, types, ptr, idx, context), y)
        kept = torch.cuda.memory_allocated() - before
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if step % 10 == 0 or step == args.steps - 1:
            say(f"step {step:4d}  loss {float(loss.detach()):.4f}  kept for backward {kept / 2 ** 20:.0f} MiB")
    return [float(v) for v in losses]


def parse(argv=None):
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("nodes", 20_000), ("features", 64), ("hidden", 128), ("classes", 8), ("experts", 8), ("top-k", 2),
                        ("steps", 60), ("seed", 0)):
        p.add_argument("--" + name, type=int, default=value)
    p.add_argument("--lr", type=float, default=3e-3)
    p.add_argument("--dtype", choices=("fp32", "fp16", "bf16"), default="fp32", help="type of the experts' rows and matrices")
    p.add_argument("--full-width", action="store_true", help="keep activations at full width")
    return p.parse_args(argv)


if __name__ == "__main__":
    run(parse())
