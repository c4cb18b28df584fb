"""What stands around the expert products of a decode step, over the C ABI.

    ScoredRouter  moe_route_scored: the experts of each token from its router logits by softmax or sigmoid
                  scores, a selection bias, expert groups, top-k, renormalised and scaled weights
    BlockNorm     moe_block_norm: the sum of a token's expert rows, the norm after the block, its gate, the
                  residual scale and add, and the norm before the next block
    Sampler       moe_sample: the next token under temperature, top-k, top-p and min-p from given uniform numbers

include/moe_prefetch.h has the formulas.  Objects hold the rule and the weights, nothing of a call: one object
may be used from several streams and threads at once.  A call launches on `stream` (a torch stream, a raw handle, or
None: the tensors' device's current stream), does not synchronise, and can be captured into a graph.  Tensors are
on one GPU; a call on another device than the current one makes it current for its length.  Outputs that are not
given are allocated on the call's stream.  Inference only: no gradients.

A decode step makes these calls in every layer, so a call is short on the host too: one pass over its arguments, its
descriptor packed at once (about 3 us before the launch itself).
"""
import torch

from . import _lib
from ._lib import MoeError, check, lib

_F32, _I32 = torch.float32, torch.int32
DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _dtype(t, what):
    d = DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    return d


def _place(t, dev, what):
    if t.device.type != "cuda":
        raise ValueError(f"{what} is on {t.device}, not on a GPU")
    raise ValueError(f"{what} is on {t.device}, the call's other tensors on cuda:{dev}")


def _on_gpu(t, what):
    """The index of t's GPU."""
    dev = t.get_device()
    if dev < 0 or not t.is_cuda:
        _place(t, dev, what)
    return dev


def _vec(t, n, dtype, dev, what):
    """The address of a contiguous vector of n elements."""
    if t.dtype is not dtype or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} vector of {n}, not {t.dtype} {tuple(t.shape)}")
    if t.get_device() != dev:
        _place(t, dev, what)
    return t.data_ptr()


def _handle(stream, dev):
    """The raw handle of a given stream: an int as it is, or a torch stream of the call's device."""
    if isinstance(stream, int):
        return stream
    if stream.device.index != dev:
        raise ValueError(f"the stream is of {stream.device}, the call's tensors on cuda:{dev}")
    return stream.cuda_stream


def _empty(shape, dtype, dev, stream):
    """Memory of the stream that the call runs on: an allocator block is safe to write on the stream it came from."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    handle = _handle(stream, dev)
    with torch.cuda.stream(torch.cuda.ExternalStream(handle, dev) if stream is handle else stream):
        return torch.empty(shape, dtype=dtype, device=dev)


def _out(t, shape, dtype, dev, what):
    """The address of a given output."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous {dtype} {shape}, not {t.dtype} {tuple(t.shape)}")
    if t.get_device() != dev:
        _place(t, dev, what)
    return t.data_ptr()


def _rows(t, rows, n, dev, what):
    """The row stride of [rows][n] with unit column stride."""
    if t.shape != (rows, n):
        raise ValueError(f"{what} must be [{rows}][{n}], not {tuple(t.shape)}")
    if t.get_device() != dev:
        _place(t, dev, what)
    ld, one = t.stride()
    if one != 1 and n > 1:
        raise ValueError(f"the columns of {what} must be next to each other, not {t.stride()} apart")
    if rows <= 1:
        return n                                      # one row: its stride is not used
    if ld < n:
        raise ValueError(f"the rows of {what} overlap (row stride {ld})")
    return ld


def _first(t, n, what):
    """(rows, row stride, device) of a call's first tensor [rows][n]."""
    if t.dim() != 2:
        raise ValueError(f"{what} must be [tokens][{n}], not {tuple(t.shape)}")
    dev, rows = _on_gpu(t, what), t.shape[0]
    return rows, _rows(t, rows, n, dev, what), dev


def _call(fn, desc, dev, stream, what):
    raw = _raw_stream(dev) if stream is None else _handle(stream, dev)
    if _device() == dev:
        rc = fn(desc, raw)
    else:
        with torch.cuda.device(dev):
            rc = fn(desc, raw)
    if rc:
        check(rc, what)


class ScoredRouter:
    """Softmax or sigmoid scores -> + bias -> groups -> top-k -> weights.

    bias: f32 [n_experts] on the GPU, added for the selection only; it is read at each call, so a balancing
    step may update it in place.  n_groups / top_groups / group_best: keep the experts of the top_groups groups
    whose best group_best (1 or 2) experts sum highest.  renormalize: divide by the sum of the chosen scores.
    """

    def __init__(self, n_experts, n_expert_used, score="softmax", bias=None, n_groups=1, top_groups=None,
                 group_best=1, renormalize=True, scale=1.0):
        if score not in _lib.SCORE:
            raise ValueError(f"score must be one of {sorted(_lib.SCORE)}, not {score!r}")
        self.E, self.K, self.bias = int(n_experts), int(n_expert_used), bias
        top = n_groups if top_groups is None else top_groups
        self._rule = (self.E, self.K, _lib.SCORE[score], int(bool(renormalize)), int(n_groups), int(top), int(group_best),
                      float(scale))
        if bias is not None:
            _vec(bias, self.E, _F32, _on_gpu(bias, "bias"), "bias")
        self._pack, self._fn = _lib.packed(_lib.RouteScoredDesc)[0], _lib.entry("moe_route_scored")
        check(self._fn(self._packed(0, 0, 0, 0), None), "moe_route_scored")     # the rule alone: no tokens

    def _packed(self, logits, ld, kind, T, bias=0, table=0, dummy=0, ids=0, w=0, slots=0, scores=0, W=0, x=0, H=0,
                workspace=0):
        return self._pack(logits, ld, kind, T, *self._rule, bias, table, dummy, ids, w, slots, scores, W, x, H, workspace)

    def rule(self):
        """The rule as a descriptor (MoeCache.set_scoring), which holds the address of the bias: whoever reads it later keeps
        that tensor."""
        bias = self.bias
        return _lib.RouteScoredDesc.from_buffer_copy(
            self._packed(0, 0, 0, 0, bias=0 if bias is None else _vec(bias, self.E, _F32, _on_gpu(bias, "bias"), "bias")))

    def from_product(self, W, x, ids, w, slots, workspace, H, stream=None):
        """The same from W [n_experts][H] and x [tokens][H] (f32), whose product moe_route's kernels make in workspace
        (BatchedMoe.route: hidden 2048, n_experts a multiple of 64 up to 256).  workspace: contiguous, of
        moe_route_workspace_bytes() at least."""
        T, _, dev = _first(x, H, "x")
        need = lib().moe_route_workspace_bytes(self.E, T)
        if workspace.nbytes < need or not workspace.is_contiguous():
            raise ValueError(f"workspace must be contiguous and of {need} bytes at least, not {tuple(workspace.shape)} of "
                             f"{workspace.dtype}")
        if workspace.get_device() != dev:
            _place(workspace, dev, "workspace")
        out = (T, self.K)
        desc = self._packed(0, 0, 0, T, 0 if self.bias is None else _vec(self.bias, self.E, _F32, dev, "bias"), 0, self.E,
                            _out(ids, out, _I32, dev, "ids"), _out(w, out, _F32, dev, "w"), _out(slots, out, _I32, dev, "slots"),
                            0, _out(W, (self.E, H), _F32, dev, "W"), _out(x, (T, H), _F32, dev, "x"), H,
                            workspace.data_ptr())
        _call(self._fn, desc, dev, stream, "moe_route_scored")

    def __call__(self, logits, ids=None, w=None, table=None, dummy=None, slots=None, scores=None, stream=None):
        """logits [tokens][n_experts] f32, bf16 or fp16 -> ids [tokens][K] int32, w [tokens][K] f32.

        slots (int32 [tokens][K]) receives table[ids] (table: int32 [n_experts]) or dummy (n_experts unless given)
        without a table; scores (f32 [tokens][n_experts]) receives every expert's score.
        """
        E, K = self.E, self.K
        T, ld, dev = _first(logits, E, "logits")
        out = (T, K)
        if ids is None:
            ids = _empty(out, _I32, dev, stream)
        if w is None:
            w = _empty(out, _F32, dev, stream)
        bias = self.bias
        desc = self._packed(logits.data_ptr(), ld, _dtype(logits, "logits"), T,
                            0 if bias is None else _vec(bias, E, _F32, dev, "bias"),
                            0 if table is None else _vec(table, E, _I32, dev, "table"), E if dummy is None else dummy,
                            _out(ids, out, _I32, dev, "ids"), _out(w, out, _F32, dev, "w"),
                            0 if slots is None else _out(slots, out, _I32, dev, "slots"),
                            0 if scores is None else _out(scores, (T, E), _F32, dev, "scores"))
        _call(self._fn, desc, dev, stream, "moe_route_scored")
        return ids, w


class BlockNorm:
    """r = x + scale * gate * post_norm(sum of the branch rows);  y = norm(r).

    weight, bias: of the norm before the next block; post_weight, post_bias: of the norm after this block, which
    is there if post (by default: if one of them is given).  All [hidden], of one dtype: f32 or x's; read at each call from
    the memory that they have now (a parameter whose data is exchanged takes another BlockNorm).  kind "rms" or "layer";
    weight_offset is added to the given weights (1 for weights stored as their distance from 1).
    """

    def __init__(self, hidden, weight=None, bias=None, post_weight=None, post_bias=None, kind="rms", eps=1e-6,
                 post_eps=None, post=None, weight_offset=0.0, scale=1.0, gate_act=None):
        if kind not in _lib.NORM:
            raise ValueError(f"kind must be one of {sorted(_lib.NORM)}, not {kind!r}")
        if gate_act not in _lib.GATE_ACT:
            raise ValueError(f"gate_act must be None or 'sigmoid', not {gate_act!r}")
        self.H = int(hidden)
        self.post = int((post_weight is not None or post_bias is not None) if post is None else bool(post))
        if not self.post and (post_weight is not None or post_bias is not None):
            raise ValueError("post-norm weights without a post-norm")
        # aliases: they keep the memory whose addresses the calls hand on, also if a parameter's data is exchanged
        self.weights = tuple(None if t is None else t.detach() for t in (weight, bias, post_weight, post_bias))
        given = [t for t in self.weights if t is not None]
        if len({t.dtype for t in given}) > 1:
            raise ValueError("the weights must be of one dtype")
        self.kind, self.act = _lib.NORM[kind], _lib.GATE_ACT[gate_act]
        self._rule = (float(scale), float(weight_offset), float(eps), float(eps if post_eps is None else post_eps))
        self._pack, self._fn = _lib.packed(_lib.BlockNormDesc)[0], _lib.entry("moe_block_norm")
        none = self._pack(0, self.H, self.kind, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, self.act, *self._rule, *[0] * 11)
        check(self._fn(none, None), "moe_block_norm")                       # the rule alone: no tokens
        self.w_dev, w_type = None, 0
        if given:
            w_type, self.w_dev = _dtype(given[0], "weight"), _on_gpu(given[0], "weight")
        names = ("weight", "bias", "post_weight", "post_bias")
        ptr = [0 if t is None else _vec(t, self.H, given[0].dtype, self.w_dev, n) for n, t in zip(names, self.weights)]
        self._w_post = (*ptr, w_type, self.post)
        self._w = (ptr[0], ptr[1], 0, 0, w_type, 0)                         # of a call without a branch

    def __call__(self, x, branch=None, gate=None, out=None, residual=None, out_dtype=None, stream=None):
        """x [tokens][hidden] f32, bf16 or fp16; branch [tokens][hidden] or [tokens][n][hidden] (its n rows are
        summed in order), f32 or x's dtype; gate [tokens], [tokens][1], [hidden] or [tokens][hidden], f32 or x's dtype
        (a vector of tokens == hidden elements is one per channel) -> (y, r).

        out receives y (of out_dtype: x's, unless given, or f32), residual receives r (x's dtype); residual=x updates
        the stream in place.  Without a branch r is x and nothing is written for it unless residual is given.
        """
        H = self.H
        T, ld, dev = _first(x, H, "x")
        dtype = x.dtype
        if self.w_dev is not None and self.w_dev != dev:
            raise ValueError(f"the weights are on cuda:{self.w_dev}, x on cuda:{dev}")
        if branch is None:
            b = (0, 0, 0, 0)
        elif branch.dim() == 3:
            n = branch.shape[1]
            b = (_out(branch, (T, n, H), branch.dtype, dev, "branch"), H, _dtype(branch, "branch"), n)
        else:
            b = (branch.data_ptr(), _rows(branch, T, H, dev, "branch"), _dtype(branch, "branch"), 1)
        if residual is not None:
            if residual.dtype is not dtype:
                raise ValueError(f"residual must be {dtype}, as x is, not {residual.dtype}")
            r = (residual.data_ptr(), _rows(residual, T, H, dev, "residual"))
        elif branch is not None:
            residual = _empty((T, H), dtype, dev, stream)
            r = (residual.data_ptr(), H)
        else:
            r = (0, 0)
        if out is None:
            out = _empty((T, H), dtype if out_dtype is None else out_dtype, dev, stream)
        elif out_dtype is not None and out.dtype is not out_dtype:
            raise ValueError(f"out is {out.dtype}, not {out_dtype}")
        desc = self._pack(T, H, self.kind, x.data_ptr(), ld, _dtype(x, "x"), *b,
                          *((0, 0, 0, 0) if gate is None else self._gate(gate, T, dev)), self.act, *self._rule,
                          *(self._w if branch is None else self._w_post), *r, out.data_ptr(),
                          _rows(out, T, H, dev, "out"), _dtype(out, "out"))
        _call(self._fn, desc, dev, stream, "moe_block_norm")
        return out, x if residual is None else residual

    def _gate(self, gate, T, dev):
        """(address, row stride, column stride, type)"""
        H, shape, at, kind = self.H, tuple(gate.shape), gate.data_ptr(), _dtype(gate, "gate")
        if gate.get_device() != dev:
            _place(gate, dev, "gate")
        if shape == (H,):
            if gate.stride(0) == 1 or H == 1:
                return at, 0, 1, kind
        elif shape == (T, H):
            return at, _rows(gate, T, H, dev, "gate"), 1, kind
        elif shape == (T,) or shape == (T, 1):
            if T <= 1 or gate.stride(0) >= 1:
                return at, gate.stride(0) if T > 1 else 1, 0, kind
        raise ValueError(f"gate must be [{T}], [{T}][1], [{H}] or [{T}][{H}], not {shape} with strides {gate.stride()}")


class Sampler:
    """The next token of each row of logits from a given uniform number."""

    def __init__(self, vocab):
        self.V = int(vocab)
        self._pack, self._fn = _lib.packed(_lib.SampleDesc)[0], _lib.entry("moe_sample")
        none = self._pack(0, 0, 0, 0, self.V, 0, 0, 0, 0, 0, 1.0, 0, 1.0, 0.0, 0, 0, 0)
        check(self._fn(none, None), "moe_sample")                           # the size alone: no tokens
        self._ws = {}                                                       # tokens -> workspace bytes

    def __call__(self, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, probs=None,
                 stream=None):
        """logits [tokens][vocab] f32, bf16 or fp16; u f32 [tokens] in [0, 1) -> tokens int32 [tokens], probs f32
        [tokens] (the share of the kept mass that the token had).

        temperature, top_p, min_p (f32) and top_k (int32): a number for every row, a tensor [tokens], or None
        (temperature 1, nothing cut).  The temperature comes before the cuts; one of 0 takes the largest logit.
        """
        V = self.V
        T, ld, dev = _first(logits, V, "logits")
        Tensor = torch.Tensor
        t_row = k_row = p_row = m_row = 0
        t_all, k_all, p_all, m_all = 1.0, 0, 1.0, 0.0
        if isinstance(temperature, Tensor):
            t_row = _vec(temperature, T, _F32, dev, "temperature")
        elif temperature is not None:
            t_all = temperature
        if isinstance(top_k, Tensor):
            k_row = _vec(top_k, T, _I32, dev, "top_k")
        elif top_k is not None:
            k_all = top_k
        if isinstance(top_p, Tensor):
            p_row = _vec(top_p, T, _F32, dev, "top_p")
        elif top_p is not None:
            p_all = top_p
        if isinstance(min_p, Tensor):
            m_row = _vec(min_p, T, _F32, dev, "min_p")
        elif min_p is not None:
            m_all = min_p
        if tokens is None:
            tokens = _empty((T,), _I32, dev, stream)
        if probs is None:
            probs = _empty((T,), _F32, dev, stream)
        size = self._ws.get(T)
        if size is None:
            if T > _lib.SAMPLE_MAX_TOKENS:
                raise MoeError(f"moe_sample: n_tok {T} out of range")
            size = self._ws[T] = lib().moe_sample_workspace_bytes(T, V)
        ws = _empty((size,), torch.uint8, dev, stream)
        desc = self._pack(logits.data_ptr(), ld, _dtype(logits, "logits"), T, V, _vec(u, T, _F32, dev, "u"), t_row, k_row,
                          p_row, m_row, t_all, k_all, p_all, m_all, _out(tokens, (T,), _I32, dev, "tokens"),
                          _out(probs, (T,), _F32, dev, "probs"), ws.data_ptr())
        _call(self._fn, desc, dev, stream, "moe_sample")
        return tokens, probs
