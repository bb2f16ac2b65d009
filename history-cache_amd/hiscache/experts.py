"""A layer of experts over the nodes of a batch, and activations kept in 8 bits for the backward pass.

``ExpertMLP`` stands behind (or in place of) the dense half of a layer: every node goes through a few of E gated maps, chosen by
a learned router or given, for instance by the node's type.  ``packed_activations`` is a context in which autograd keeps
what operators save in 8 bits.  Both run on ``hiscache_backend``'s kernels.
"""
import math

import torch
import torch.nn.functional as F

import hiscache_backend


class ExpertMLP(torch.nn.Module):
    """``sum_j weight[i, j] * expert[i, j](x[i])`` with ``expert_e(x) = (silu(x A_e) * (x B_e)) C_e``.

    channels: width of the rows in and out; hidden: width inside an expert; num_expert: E; top_k: experts a row;
    normalize: a row's weights add up to one.  In training [x A | x B] is kept in 8 bits, a scale for every ``group`` columns."""

    def __init__(self, channels, hidden, num_expert, top_k=2, normalize=True, group=64, device=None, dtype=None):
        super().__init__()
        if not 1 <= top_k <= num_expert:
            raise ValueError(f"top_k must be between 1 and the {num_expert} experts, got {top_k}")
        self.channels, self.hidden, self.num_expert = channels, hidden, num_expert
        self.top_k, self.normalize, self.group = top_k, normalize, group
        # the router's logits are fp32 whatever the rows are, under autocast and in a module cast to half precision as well: near-ties
        # decide where a row goes
        self.router = torch.nn.Parameter(torch.empty(num_expert, channels, device=device, dtype=torch.float32))
        self.w_in = torch.nn.Parameter(torch.empty(num_expert, 2 * hidden, channels, device=device, dtype=dtype))
        self.w_out = torch.nn.Parameter(torch.empty(num_expert, channels, hidden, device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            for w, fan in ((self.router, self.channels), (self.w_in, self.channels), (self.w_out, self.hidden)):
                w.uniform_(-1 / math.sqrt(fan), 1 / math.sqrt(fan))

    def route(self, x, allowed=None):
        """The router's choice for the rows of x: (expert int64 [n, top_k], weight fp32 [n, top_k]).  ``allowed`` (bool
        [n, E] or [E], optional): experts that a row may go to; a row that may go nowhere gets -1 and weight 0."""
        if torch.is_autocast_enabled(x.device.type):
            with torch.autocast(x.device.type, enabled=False):
                logits = F.linear(x.float(), self.router.float())
        else:
            logits = F.linear(x.float(), self.router.float())
        if allowed is not None:
            logits = logits.masked_fill(~allowed, -math.inf)
        return hiscache_backend.route_rows(logits, self.top_k, normalize=self.normalize)

    def forward(self, x, expert=None, weight=None, allowed=None):
        """x [n, channels] through its experts.  ``expert`` (int64 [n] or [n, k]) and ``weight`` (fp32, default ones) replace
        the router's choice; -1 sends a row nowhere (zeros, if it has no other).  ``allowed`` is for the router
        (:meth:`route`)."""
        be = hiscache_backend
        if (weight if expert is None else allowed) is not None:
            raise ValueError("weight goes with expert, allowed with the router's choice")
        if expert is None:
            expert, weight = self.route(x, allowed)
        order = be.expert_order(expert, self.num_expert)
        y = be.gated_experts(be.rows_to_experts(x, order), self.w_in, self.w_out, order.offset, self.group)
        return be.rows_from_experts(y, order, weight)

    def extra_repr(self):
        return (f"{self.channels}, hidden={self.hidden}, num_expert={self.num_expert}, top_k={self.top_k}, "
                f"normalize={self.normalize}, group={self.group}")


# Steps back through the history of a matrix that are looked at: a cast, a slice or a normalised weight is up to six from its
# parameter, a stack of weights with an update of low rank ten (twelve take the host about as long as packing).
_WEIGHT_STEPS = 12


def _result_shape(node, i):
    """The shape of a node's i-th result."""
    leaf = getattr(node, "variable", None)
    return tuple(leaf.shape if leaf is not None else node._input_metadata[i].shape)


def _is_weight(t):
    """Is t a parameter or a leaf that needs a gradient, a view of one, or computed from parameters alone?  The last is told by t's
    history: it ends at parameters within a few steps, and no data took part in it -- an index, or an operand that needs no
    gradient in a step whose result has another shape than the other operand (rows of a batch; a number has none) --, or t has
    as many elements as one of the parameters all the same."""
    base = t if t._base is None else t._base
    if isinstance(base, torch.nn.Parameter) or (base.is_leaf and base.requires_grad):
        return True
    if t.grad_fn is None:
        return False
    nodes, data, alike = [(t.grad_fn, 0)], False, False
    for _ in range(_WEIGHT_STEPS):
        if not nodes:
            break
        node, i = nodes.pop()
        if isinstance(node, torch.autograd.function.BackwardCFunction):
            return False                                  # an operator of its own, whatever it takes
        leaf = getattr(node, "variable", None)
        if leaf is not None:
            if not isinstance(leaf, torch.nn.Parameter):
                return False
            alike = alike or leaf.numel() == t.numel()
            continue
        before = [edge for edge in node.next_functions if edge[0] is not None]
        if node.name().startswith(("Embedding", "Index", "Gather")):
            data = True
        elif len(before) < len(node.next_functions):
            if any(isinstance(n, torch.autograd.function.BackwardCFunction) for n, _ in before):
                return False
            data = data or _result_shape(node, i) not in [_result_shape(*edge) for edge in before]
        nodes += before
    return not nodes and (alike or not data)


def _is_activation(t, min_elements, group=64):
    """Is what autograd saves here a matrix that may be kept in 8 bits, and does it get smaller (a narrow row's scales weigh more
    than what its values lose)?"""
    return (t.layout is torch.strided and t.dtype in hiscache_backend._DTYPES and t.dim() >= 2 and t.numel() >= max(min_elements, 1)
            and t.shape[-1] + 4 * -(-t.shape[-1] // group) < t.shape[-1] * t.element_size()
            and t.is_contiguous() and not _is_weight(t))


def packed_activations(group=64, min_elements=1 << 16):
    """Context in which what autograd saves for backward is kept in 8 bits, a scale for every ``group`` columns
    (``hiscache_backend.pack_rows``): the gradients are those at activations that are off by up to half a scale
    (16-bit ones by what they are rounded to their type besides: up to a whole scale in bf16).

    Kept as they are: parameters, views of parameters and matrices computed from parameters alone in a few steps (a cast copy,
    a scaled or normalised weight); other leaves that need a gradient and their views; whole numbers; tensors of fewer than
    ``min_elements`` values, without a last dimension of their own or so narrow that codes and scales would not be smaller;
    sparse tensors; and anything not packed in the current GPU's memory.  Any other matrix counts as an activation, a copy of a
    frozen weight among them, since nothing tells it from the rows of a batch: run a product by one outside.  A matrix that
    several operators save is kept once for each of them, and one that the caller holds on to is kept besides.  Put the context
    around the layers whose activations may be rounded; a loss, a softmax, attention (whose sums of exponentials would be rounded as
    logarithms) or the router's weights are better left outside."""
    be = hiscache_backend

    def pack(t):
        if not t.is_cuda or t.device.index != torch.cuda.current_device() or not _is_activation(t, min_elements, group):
            # (a node that held its own result would be held by it in turn, out of the garbage collector's sight)
            t = t if t.is_leaf else t.detach()
            return t, t._version
        return be.pack_rows(t.detach().view(-1, t.shape[-1]), group), t.shape

    def unpack(saved):
        kept, of = saved
        if not isinstance(kept, torch.Tensor):
            return be.unpack_rows(kept).view(of)
        # (autograd itself looks at versions only where there are no hooks)
        if kept._version != of:
            raise RuntimeError("one of the variables needed for gradient computation has been modified by an inplace operation: "
                               f"{kept.dtype} {list(kept.shape)} is at version {kept._version}; expected version {of} instead")
        return kept

    return torch.autograd.graph.saved_tensors_hooks(pack, unpack)
