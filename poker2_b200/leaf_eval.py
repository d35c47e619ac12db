"""Leaf evaluators for subgames that end before the river: the callables a `SteppedSolver`
invokes between the two sweeps of every pass.

Upstream, the leaves at the start of the next street are valued by the value network
(`set_leaf_values`, p2/search/cfr_evaluator.py:1025-1047), and the value of such a
pre-chance state is the expectation over the next public card of the network's values on
the post-card beliefs (`ChanceNodeHelper.single_card_chance_values`,
p2/search/chance_node_helper.py:359-479).  `ChanceLeafEvaluator` computes that expectation
explicitly: the expansion over the next card and the per-leaf averaging are this library's
kernels (`chance.expand_next_card`, `chance.indexed_add_rows`); the GEMMs of `ValueMLP` are
torch / cuBLAS, `GatedValueMLP` and `Mx4ValueMLP` are made of this library's gated and 4-bit
layers.
"""
from __future__ import annotations

import copy
import threading

import numpy as np
import torch

from . import _lib, chance, gated, mx4

NUM_HANDS = 1326


class ValueMLP(torch.nn.Module):
    """Value network stand-in with the shape of the benchmark configuration: input = two
    1326-combo ranges + 52-d board one-hot + 3 pot/stack scalars, `depth` hidden layers of
    `width` GELU units, output = 2 x 1326 hand values.  Random initialisation."""

    IN_FEATURES = 2 * NUM_HANDS + 52 + 3  # 2707
    IN_PADDED = 2720  # GEMM operands want rows that are multiples of 16 bytes; the extra columns are zero
    OUT_PADDED = 2656

    def __init__(self, width: int = 1536, depth: int = 4, *, dtype=torch.bfloat16, seed: int = 0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        dims = [self.IN_FEATURES] + [width] * depth + [2 * NUM_HANDS]
        padded = [self.IN_PADDED] + [width] * depth + [self.OUT_PADDED]
        layers = []
        for i in range(len(dims) - 1):
            lin = torch.nn.Linear(padded[i], padded[i + 1])
            with torch.no_grad():
                lin.weight.zero_()
                lin.weight[: dims[i + 1], : dims[i]] = torch.randn(dims[i + 1], dims[i], generator=g) / dims[i] ** 0.5
                lin.bias.zero_()
            layers.append(lin)
            if i < len(dims) - 2:
                layers.append(torch.nn.GELU())
        self.net = torch.nn.Sequential(*layers).to(dtype)
        self.dtype = dtype

    @torch.no_grad()
    def forward(self, beliefs: torch.Tensor, boards: torch.Tensor, context: torch.Tensor) -> torch.Tensor:
        """beliefs [S,2,1326] fp32, boards [S,L] int64 (-1 = empty), context [S,3] fp32
        -> values [S,2,1326] fp32."""
        S = beliefs.shape[0]
        x = torch.zeros(S, self.IN_PADDED, device=beliefs.device, dtype=self.dtype)
        x[:, : 2 * NUM_HANDS] = beliefs.reshape(S, 2 * NUM_HANDS)
        onehot = torch.zeros(S, 53, device=beliefs.device, dtype=self.dtype)
        onehot.scatter_(1, torch.where(boards >= 0, boards, torch.full_like(boards, 52)), 1.0)
        x[:, 2 * NUM_HANDS: 2 * NUM_HANDS + 52] = onehot[:, :52]
        x[:, 2 * NUM_HANDS + 52: self.IN_FEATURES] = context
        y = self.net(x)[:, : 2 * NUM_HANDS]
        return y.to(torch.float32).view(S, 2, NUM_HANDS)

    @torch.no_grad()
    def layers(self, x: torch.Tensor) -> torch.Tensor:
        """`self.net` on input rows x, activations in place (half the memory traffic and footprint of a GELU, same bits) and
        linear layers without the module's wrapper: a pass over few leaves lasts as long as the host takes to launch it.
        A network that someone listens to (hooks) or has changed goes through its modules instead."""
        net = self.net
        if type(net) is not torch.nn.Sequential or not _bare(net, *net._modules.values()):
            return net(x)
        for layer in net._modules.values():
            if type(layer) is torch.nn.GELU and layer.approximate == "none":
                x = torch.ops.aten.gelu_(x)
            elif type(layer) is torch.nn.Linear:
                x = torch.nn.functional.linear(x, layer.weight, layer.bias)
            else:
                x = layer(x)
        return x


class GatedBlock(torch.nn.Module):
    """x + Wd (act(Wg n(x) + bg) * (Wu n(x) + bu)) + bd with n a layer norm: the gated hidden layer as a residual block.  `keep`: as in
    `gated.gated_linear`."""

    def __init__(self, width: int, hidden: int, *, activation: str = "gelu", keep: bool = True, generator: torch.Generator | None = None):
        super().__init__()
        self.norm = torch.nn.LayerNorm(width)
        new = lambda rows, columns: torch.nn.Parameter(torch.randn(rows, columns, generator=generator) / columns ** 0.5)  # noqa: E731
        self.gate_weight, self.up_weight = new(hidden, width), new(hidden, width)
        self.gate_bias, self.up_bias = torch.nn.Parameter(torch.zeros(hidden)), torch.nn.Parameter(torch.zeros(hidden))
        self.down = torch.nn.Linear(hidden, width)
        with torch.no_grad():
            self.down.weight.copy_(new(width, hidden))
            self.down.bias.zero_()
        self.activation, self.keep = activation, keep

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = gated.gated_linear(self.norm(x), self.gate_weight, self.up_weight, self.gate_bias, self.up_bias, activation=self.activation, keep=self.keep)
        return x + self.down(h)


class GatedValueMLP(ValueMLP):
    """`ValueMLP` with `depth - 1` gated residual blocks of `hidden` units for its inner layers; same input and output rows, so
    the leaf evaluators take it on the same paths.  Runs on the GPU, bf16 or fp16."""

    def __init__(self, width: int = 1536, depth: int = 4, *, hidden: int | None = None, activation: str = "gelu", keep: bool = True, dtype=torch.bfloat16, seed: int = 0):
        super().__init__(width, 1, dtype=dtype, seed=seed)
        g = torch.Generator().manual_seed(seed + 1)
        first, act, last = self.net
        blocks = [GatedBlock(width, hidden or 2 * width // 3, activation=activation, keep=keep, generator=g) for _ in range(depth - 1)]
        self.net = torch.nn.Sequential(first, act, *blocks, last).to(dtype)


def _refuse_type_change(fn, dtype: torch.dtype, device: torch.device) -> None:
    if fn(torch.empty(0, dtype=dtype, device=device)).dtype != dtype:
        raise ValueError("a 4-bit layer or network keeps its type: quantise a source of the other one")


class Mx4Linear(torch.nn.Module):
    """act(q(x) q(W)^T + b) with W quantised once, when the layer is made.  `hands_on`: the result stays in 4 bits, as the next such
    layer would make of it (but for few rows, which that one takes as they are).  W is in the state dict in 4 bits; the layer moves
    between devices and keeps its type."""

    def __init__(self, linear: torch.nn.Linear, activation: str = "none", hands_on: bool = False):
        super().__init__()
        weight = mx4.quantise(linear.weight.detach())
        self.register_buffer("values", weight.values)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().clone())
        self.shape = weight.shape
        self.activation, self.hands_on, self.dtype = activation, hands_on, linear.weight.dtype

    @property
    def weight(self) -> mx4.Mx4:
        own, m = self._buffers, self.__dict__.get("_weight")
        if m is None or m.values is not own["values"] or m.scales is not own["scales"]:
            m = self.__dict__["_weight"] = mx4.Mx4(own["values"], own["scales"], self.shape)
        return m

    def forward(self, x: torch.Tensor | mx4.Mx4) -> torch.Tensor | mx4.Mx4:
        rows = x.rows if isinstance(x, mx4.Mx4) else x.shape[:-1].numel()
        return mx4.linear(x, self.weight, self.bias, activation=self.activation, dtype=self.dtype, quantised=self.hands_on and rows > mx4.FEW_ROWS)

    def _apply(self, fn, recurse=True):
        _refuse_type_change(fn, self.dtype, self.values.device)
        self.__dict__.pop("_weight", None)  # (it holds the arrays that are left behind)
        return super()._apply(fn, recurse)

    def get_extra_state(self):  # (widths up to 31 apart have arrays of one size)
        return {"shape": self.shape}

    def set_extra_state(self, state):
        pass

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        saved = state_dict.get(prefix + "_extra_state")
        if saved is not None and tuple(saved["shape"]) != self.shape:
            error_msgs.append(f"a 4-bit weight of {tuple(saved['shape'])} does not fit {prefix[:-1] or 'the layer'}, whose weight is {self.shape}")
            return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)


class Mx4ValueMLP(ValueMLP):
    """A `ValueMLP` as it serves in 4 bits: every linear layer with its GELU becomes an `Mx4Linear`.  A copy of the weights as
    they are now, on the GPU where they lie, saved and moved as other networks are; for leaf values, not for training.

    What it costs: with random weights and a width of 1536 the values of 4096 leaves lie 26 % of their norm from the source's in
    fp32 with two hidden layers and 35 % with four (bf16: 0.4 and 0.5 %); each layer adds 12 % for its weights and about as much for its
    input.  The input rows fare worse than that where a block of 32 columns holds unlike things: while one of cards 0 to 3 lies on the
    board, entries below 1/16 among the second player's last 28 hands count as 0, and while one of cards 36 to 51 does, pot and stacks
    are in eighths (quarters from 1/2 on); the same goes for the weights of these columns.  `quantise_first=False` leaves the first layer
    in 16 bits: where its weights on the ranges are 30 times the others, 32 % instead of 50 % with four hidden layers and a low card."""

    def __init__(self, source: ValueMLP, *, quantise_first: bool = True):
        torch.nn.Module.__init__(self)
        if type(source) is not ValueMLP:
            raise ValueError("a bf16 or fp16 ValueMLP is quantised")
        layers = list(source.net)
        # (of the layers themselves: a source that was turned into another type still says the one it was made in)
        types = {t.dtype for t in source.net.parameters()}
        if len(types) != 1 or not types <= {torch.bfloat16, torch.float16}:
            raise ValueError("a bf16 or fp16 ValueMLP is quantised, all its layers of one type")
        if any(type(m) not in (torch.nn.Linear, torch.nn.GELU) or type(m) is torch.nn.GELU and m.approximate != "none" for m in layers):
            raise ValueError("linear layers and GELUs are quantised, nothing else")
        if any(type(m) is torch.nn.GELU and (i == 0 or type(layers[i - 1]) is not torch.nn.Linear) for i, m in enumerate(layers)):
            raise ValueError("a GELU follows a linear layer")
        after = lambda i: "gelu" if i + 1 < len(layers) and type(layers[i + 1]) is torch.nn.GELU else "none"  # noqa: E731
        last = max(i for i, m in enumerate(layers) if type(m) is torch.nn.Linear)
        if last == 0 and not quantise_first:
            raise ValueError("a network of one layer has nothing else to quantise")
        quantised = [Mx4Linear(m, after(i), i < last) for i, m in enumerate(layers) if type(m) is torch.nn.Linear and (quantise_first or i > 0)]
        kept = [] if quantise_first else [copy.deepcopy(layers[0]).requires_grad_(False)] + [torch.nn.GELU()] * (after(0) == "gelu")
        self.net = torch.nn.Sequential(*kept, *quantised)
        self.dtype = types.pop()

    def _apply(self, fn, recurse=True):
        _refuse_type_change(fn, self.dtype, next(self.buffers()).device)  # (before any layer is changed)
        return super()._apply(fn, recurse)


# networks whose input and output rows are those of `ValueMLP`
_ROW_NETWORKS = (ValueMLP, GatedValueMLP, Mx4ValueMLP)
_module_hooks = torch.nn.modules.module


def _bare(*modules: torch.nn.Module) -> bool:
    """Nothing but the modules' own `forward` would run if they were called: no forward hooks, on them or on all modules, no
    `forward` put in place of the class's, not compiled.  (By their dictionaries: asked once a pass, for nine modules.)"""
    if _module_hooks._global_forward_hooks or _module_hooks._global_forward_pre_hooks:
        return False
    for m in modules:
        own = m.__dict__
        if own["_forward_hooks"] or own["_forward_pre_hooks"] or "forward" in own or own.get("_compiled_call_impl") is not None:
            return False
    return True


def leaf_context(trees, node_index) -> torch.Tensor:
    """[L,3] fp32 context of the tree nodes `node_index` (upstream numbering): pot and both
    stacks as fractions of the two starting stacks together."""
    st = trees.state
    idx = np.asarray(node_index, dtype=np.int64)
    total = np.maximum(st.starting_stacks[idx].astype(np.float32).sum(axis=1), np.float32(1.0))
    f32 = lambda a: a.astype(np.float32)  # noqa: E731  (fp32 division, as the upstream encoder does)
    ctx = np.stack([f32(st.pot[idx]) / total, f32(st.stacks[idx, 0]) / total, f32(st.stacks[idx, 1]) / total], axis=1)
    return torch.from_numpy(np.ascontiguousarray(ctx, dtype=np.float32))


class ChanceLeafEvaluator:
    """values(leaf) = mean over the next public card of model(post-card beliefs).

    boards: [L,W] int64 public cards of each leaf with -1 in the empty slots (at least one);
    context: [L,3] fp32; model(beliefs [S,2,1326], boards [S,W], context [S,3]) -> [S,2,1326].
    Leaves are processed `chunk` at a time (a chunk expands to about 48 x chunk samples)."""

    def __init__(self, model, boards: torch.Tensor, context: torch.Tensor, device: torch.device, *, chunk: int = 2048):
        self.model = model
        self.boards = boards.to(device=device, dtype=torch.int64).contiguous()
        self.context = context.to(device=device, dtype=torch.float32).contiguous()
        self.chunk = int(chunk)
        self.samples_per_call = int((52 - (self.boards >= 0).sum(dim=1)).sum().item())
        self.calls = 0
        # a bf16 `ValueMLP` takes the fused path: the network input is written directly by the
        # expansion kernel and its bf16 output is averaged per leaf without an fp32 copy
        self.fused = isinstance(model, ValueMLP) and model.dtype == torch.bfloat16
        self._chunks = []
        for a in range(0, self.boards.shape[0], self.chunk):
            b = min(a + self.chunk, self.boards.shape[0])
            off = chance.sample_offsets_of(self.boards[a:b])
            self._chunks.append((a, b, off, int(off[-1].item())))

    def evaluate_into(self, leaf_beliefs: torch.Tensor, out: torch.Tensor) -> None:
        """Values of all leaves into out[..., :1326] (fp32 [L,2,W])."""
        if not self.fused:
            out[..., :NUM_HANDS].copy_(self(leaf_beliefs))
            return
        for a, b, off, n_samples in self._chunks:
            x = chance.expand_features_bf16(leaf_beliefs[a:b], self.boards[a:b], off, n_samples, self.context[a:b],
                                            self.model.IN_PADDED)
            y = self.model.layers(x)
            chance.indexed_mean_bf16(y, off, out[a:b])
        self.calls += 1

    def __call__(self, leaf_beliefs: torch.Tensor) -> torch.Tensor:
        L = leaf_beliefs.shape[0]
        if self.fused:
            out = torch.zeros(L, 2, leaf_beliefs.shape[2], device=leaf_beliefs.device, dtype=torch.float32)
            self.evaluate_into(leaf_beliefs, out)
            return out
        out = torch.empty(L, 2, NUM_HANDS, device=leaf_beliefs.device, dtype=torch.float32)
        for a in range(0, L, self.chunk):
            b = min(a + self.chunk, L)
            pre = leaf_beliefs[a:b, :, :NUM_HANDS].contiguous()
            ctx = self.context[a:b]
            out[a:b] = chance.single_card_chance_values(
                pre, self.boards[a:b], lambda post, samples, lookup: self.model(post, samples, ctx[lookup]))
        self.calls += 1
        return out


class DirectLeafEvaluator:
    """values(leaf) = model(beliefs at the leaf): the network is trained to predict the
    pre-chance value itself, which is how the upstream CFR loop calls it."""

    def __init__(self, model, boards: torch.Tensor, context: torch.Tensor, device: torch.device):
        self.model = model
        self.boards = boards.to(device=device, dtype=torch.int64).contiguous()
        self.context = context.to(device=device, dtype=torch.float32).contiguous()

        # a bf16 `ValueMLP` reads rows that the feature kernel writes: the columns that no pass changes (board
        # one-hot, context, padding) are filled in once
        self._rows = None
        self._rows_lock = threading.RLock()
        if type(model) in _ROW_NETWORKS and model.dtype == torch.bfloat16 and self.boards.is_cuda and self.boards.shape[0] > 0:
            L, first = self.boards.shape[0], 2 * NUM_HANDS
            x = torch.zeros(L, ValueMLP.IN_PADDED, device=device, dtype=torch.bfloat16)
            card = torch.arange(52, device=device)
            x[:, first: first + 52] = (self.boards[:, :, None] == card).any(dim=1)
            x[:, first + 52: ValueMLP.IN_FEATURES] = self.context
            self._rows = x
            self._rows_stream = _lib.stream_ptr(x.device)  # where the rows are at home

    def evaluate_into(self, leaf_beliefs: torch.Tensor, out: torch.Tensor) -> None:
        """Values of all leaves into out[..., :1326] (fp32 [L,2,W])."""
        if not (self._direct() and _paired_rows(leaf_beliefs, self._rows) and _paired_rows(out, self._rows)):
            out[..., :NUM_HANDS].copy_(self.model(leaf_beliefs[..., :NUM_HANDS].contiguous(), self.boards, self.context))
            return
        p, L = _lib.ptr, leaf_beliefs.shape[0]
        # calls from several threads take the rows in turn, calls on another stream (or recorded for later) a copy of them
        with _lib.on(out.device), torch.no_grad(), self._rows_lock:
            stream, rows = _lib.stream_ptr(out.device), self._rows
            if stream != self._rows_stream:
                rows = rows.clone()
                if not torch.cuda.is_current_stream_capturing():
                    self._rows.record_stream(torch.cuda.current_stream(out.device))
            _lib.call("p2b_leaf_features_bf16", p(leaf_beliefs), leaf_beliefs.stride(1), L, p(rows), rows.stride(0), stream)
            y = self.model.layers(rows)
            _lib.call("p2b_leaf_values_bf16", p(y), y.stride(0), L, p(out), out.stride(1), stream)

    def __getstate__(self):  # (a lock is neither copied nor pickled)
        return {k: v for k, v in self.__dict__.items() if k != "_rows_lock"}

    def __setstate__(self, state):
        self.__dict__.update(state, _rows_lock=threading.RLock())

    def _direct(self) -> bool:
        """The model's layers may be called on rows kept here instead of the model itself."""
        return self._rows is not None and type(self.model) in _ROW_NETWORKS and self.model.dtype == torch.bfloat16 and _bare(self.model)

    def __call__(self, leaf_beliefs: torch.Tensor) -> torch.Tensor:
        if not self._direct():
            return self.model(leaf_beliefs[..., :NUM_HANDS].contiguous(), self.boards, self.context)
        out = torch.empty(leaf_beliefs.shape[0], 2, NUM_HANDS, device=leaf_beliefs.device, dtype=torch.float32)
        self.evaluate_into(leaf_beliefs, out)
        return out


def _paired_rows(t: torch.Tensor, network_rows: torch.Tensor) -> bool:
    """[L,2,W] fp32, rows of whole pairs of hands one after the other, as many leaves as there are network rows."""
    if t.dim() != 3 or t.dtype != torch.float32 or t.device != network_rows.device:
        return False
    leaves, players, width = t.shape
    per_leaf, per_player, per_hand = t.stride()
    return (leaves == network_rows.shape[0] and players == 2 and width >= NUM_HANDS and per_hand == 1
            and per_leaf == 2 * per_player and per_player % 2 == 0 and t.data_ptr() % 8 == 0)
