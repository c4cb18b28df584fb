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
"""
import ctypes

import torch

from . import _lib
from ._lib import check, lib

DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_RAW_STREAM = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _dtype(t, what):
    d = DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    return d


def _on(t, dev, what):
    if t.device != dev or t.device.type != "cuda":
        raise ValueError(f"{what} is on {t.device}, not on a GPU" if t.device.type != "cuda"
                         else f"{what} is on {t.device}, the call's other tensors on {dev}")


def _vec(t, n, dtype, dev, what):
    """A contiguous vector of n elements: its address, or None."""
    if t is None:
        return None
    if t.dtype is not dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} vector of {n}, not {t.dtype} {tuple(t.shape)}")
    _on(t, dev, what)
    return t.data_ptr()


def _empty(shape, dtype, dev, stream):
    """Memory of the stream that the call runs on: an allocator block is safe to write on the stream it came from."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, dev) if isinstance(stream, int) else stream):
        return torch.empty(shape, dtype=dtype, device=dev)


def _out(t, shape, dtype, dev, what, stream=None):
    if t is None:
        return _empty(shape, dtype, dev, stream)
    if t.dtype is not dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous {dtype} {shape}, not {t.dtype} {tuple(t.shape)}")
    _on(t, dev, what)
    return t


def _rows(t, n, dev, what):
    """[rows][n] with unit column stride: its row stride."""
    if t.dim() != 2 or t.shape[1] != n or (n > 1 and t.stride(1) != 1):
        raise ValueError(f"{what} must be [tokens][{n}] with its columns next to each other, "
                         f"not {tuple(t.shape)} with strides {t.stride()}")
    _on(t, dev, what)
    ld = t.stride(0)
    if t.shape[0] <= 1:
        return n                                      # one row: its stride is not used
    if ld < n:
        raise ValueError(f"the rows of {what} overlap (row stride {ld})")
    return ld


def _call(fn, desc, dev, stream, what):
    if stream is None:
        raw = _RAW_STREAM(dev.index) if _RAW_STREAM else torch.cuda.current_stream(dev).cuda_stream
    else:
        raw = stream if isinstance(stream, int) else stream.cuda_stream
    if torch.cuda.current_device() == dev.index:
        check(fn(ctypes.byref(desc), raw), what)
    else:
        with torch.cuda.device(dev):
            check(fn(ctypes.byref(desc), raw), what)


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
        self._desc = _lib.RouteScoredDesc(n_tok=0, E=self.E, K=self.K, score=_lib.SCORE[score],
                                          renormalize=int(bool(renormalize)), n_groups=int(n_groups),
                                          top_groups=int(top), group_best=int(group_best), scale=float(scale))
        if bias is not None:
            _vec(bias, self.E, torch.float32, bias.device, "bias")
        check(lib().moe_route_scored(ctypes.byref(self._desc), None), "moe_route_scored")   # the rule alone: n_tok 0

    def __call__(self, logits, ids=None, w=None, table=None, dummy=None, slots=None, scores=None, stream=None):
        """logits [tokens][n_experts] f32, bf16 or fp16 -> ids [tokens][K] int32, w [tokens][K] f32.

        slots (int32 [tokens][K]) receives table[ids] (table: int32 [n_experts]) or dummy (n_experts unless given)
        without a table; scores (f32 [tokens][n_experts]) receives every expert's score.
        """
        dev = logits.device
        d = _lib.RouteScoredDesc.from_buffer_copy(self._desc)
        d.logits_type = _dtype(logits, "logits")
        d.logits_stride = _rows(logits, self.E, dev, "logits")
        T = logits.shape[0]
        ids = _out(ids, (T, self.K), torch.int32, dev, "ids", stream)
        w = _out(w, (T, self.K), torch.float32, dev, "w", stream)
        d.logits, d.n_tok, d.ids, d.w = logits.data_ptr(), T, ids.data_ptr(), w.data_ptr()
        if self.bias is not None:
            d.bias = _vec(self.bias, self.E, torch.float32, dev, "bias")
        if table is not None:
            d.table = _vec(table, self.E, torch.int32, dev, "table")
        d.dummy = self.E if dummy is None else dummy
        if slots is not None:
            d.slots = _out(slots, (T, self.K), torch.int32, dev, "slots").data_ptr()
        if scores is not None:
            d.scores = _out(scores, (T, self.E), torch.float32, dev, "scores").data_ptr()
        _call(lib().moe_route_scored, d, dev, stream, "moe_route_scored")
        return ids, w


class BlockNorm:
    """r = x + scale * gate * post_norm(sum of the branch rows);  y = norm(r).

    weight, bias: of the norm before the next block; post_weight, post_bias: of the norm after this block, which
    is there if post (by default: if one of them is given).  All [hidden], of one dtype: f32 or x's.  kind "rms" or "layer";
    weight_offset is added to the given weights (1 for weights stored as their distance from 1).
    """

    def __init__(self, hidden, weight=None, bias=None, post_weight=None, post_bias=None, kind="rms", eps=1e-6,
                 post_eps=None, post=None, weight_offset=0.0, scale=1.0, gate_act=None):
        if kind not in _lib.NORM:
            raise ValueError(f"kind must be one of {sorted(_lib.NORM)}, not {kind!r}")
        if gate_act not in _lib.GATE_ACT:
            raise ValueError(f"gate_act must be None or 'sigmoid', not {gate_act!r}")
        self.H = int(hidden)
        self.post = (post_weight is not None or post_bias is not None) if post is None else bool(post)
        if not self.post and (post_weight is not None or post_bias is not None):
            raise ValueError("post-norm weights without a post-norm")
        self.weights = (weight, bias, post_weight, post_bias)
        given = [t for t in self.weights if t is not None]
        if len({t.dtype for t in given}) > 1:
            raise ValueError("the weights must be of one dtype")
        self.w_dtype = given[0].dtype if given else torch.float32
        self.w_dev = given[0].device if given else None
        d = _lib.BlockNormDesc(n_tok=0, H=self.H, kind=_lib.NORM[kind], gate_act=_lib.GATE_ACT[gate_act],
                               scale=float(scale), weight_offset=float(weight_offset), eps=float(eps),
                               post_eps=float(eps if post_eps is None else post_eps))
        if given:
            _dtype(given[0], "weight")
        check(lib().moe_block_norm(ctypes.byref(d), None), "moe_block_norm")        # the rule alone: n_tok 0
        names = ("weight", "bias", "post_weight", "post_bias")
        for name, t in zip(names, self.weights):
            if t is not None:
                setattr(d, name, _vec(t, self.H, self.w_dtype, self.w_dev, name))
        self._desc = d

    def __call__(self, x, branch=None, gate=None, out=None, residual=None, out_dtype=None, stream=None):
        """x [tokens][hidden] f32, bf16 or fp16; branch [tokens][hidden] or [tokens][n][hidden] (its n rows are
        summed in order), f32 or x's dtype; gate [tokens], [tokens][1], [hidden] or [tokens][hidden], f32 or x's dtype
        (a vector of tokens == hidden elements is one per channel) -> (y, r).

        out receives y (of out_dtype: x's, unless given, or f32), residual receives r (x's dtype); residual=x updates
        the stream in place.  Without a branch r is x and nothing is written for it unless residual is given.
        """
        dev, H = x.device, self.H
        d = _lib.BlockNormDesc.from_buffer_copy(self._desc)
        d.x_type = _dtype(x, "x")
        d.x_stride = _rows(x, H, dev, "x")
        T = x.shape[0]
        d.n_tok, d.x = T, x.data_ptr()
        if self.w_dev is not None:
            if self.w_dev != dev:
                raise ValueError(f"the weights are on {self.w_dev}, x on {dev}")
            d.weight_type = DTYPES[self.w_dtype]
        if branch is not None:
            d.branch_type = _dtype(branch, "branch")
            d.post = int(self.post)
            if branch.dim() == 3:
                n = branch.shape[1]
                if branch.shape[0] != T or branch.shape[2] != H or not branch.is_contiguous():
                    raise ValueError(f"branch must be contiguous [{T}][n][{H}], not {tuple(branch.shape)}")
                _on(branch, dev, "branch")
                d.branch_stride, d.n_sum = H, n
            else:
                d.branch_stride, d.n_sum = _rows(branch, H, dev, "branch"), 1
                if branch.shape[0] != T:
                    raise ValueError(f"branch has {branch.shape[0]} rows, x {T}")
            d.branch = branch.data_ptr()
        if gate is not None:
            self._gate(d, gate, T, dev)
        if residual is None and branch is not None:
            residual = _empty((T, H), x.dtype, dev, stream)
        if residual is not None:
            if residual.dtype is not x.dtype or residual.shape[0] != T:
                raise ValueError(f"residual must be {x.dtype} [{T}][{H}]")
            d.residual_stride = _rows(residual, H, dev, "residual")
            d.residual = residual.data_ptr()
        if out is None:
            out = _empty((T, H), x.dtype if out_dtype is None else out_dtype, dev, stream)
        elif out.shape[0] != T or (out_dtype is not None and out.dtype is not out_dtype):
            raise ValueError(f"out must be {out_dtype or out.dtype} [{T}][{H}]")
        d.y_type = _dtype(out, "out")
        d.y_stride = _rows(out, H, dev, "out")
        d.y = out.data_ptr()
        _call(lib().moe_block_norm, d, dev, stream, "moe_block_norm")
        return out, x if residual is None else residual

    def _gate(self, d, gate, T, dev):
        H = self.H
        _on(gate, dev, "gate")
        d.gate_type = _dtype(gate, "gate")
        shape = tuple(gate.shape)
        if shape == (H,):
            row, col = 0, 1
        elif shape == (T,) or shape == (T, 1):
            row, col = 1, 0
        elif shape == (T, H):
            row, col = H, 1
        else:
            raise ValueError(f"gate must be [{T}], [{T}][1], [{H}] or [{T}][{H}], not {shape}")
        if col and H > 1 and gate.stride(-1) != 1:
            raise ValueError(f"the columns of gate must be next to each other, not {gate.stride()}")
        if row and T > 1:
            row = gate.stride(0)
            if row < (H if col else 1):
                raise ValueError(f"the rows of gate overlap (row stride {row})")
        d.gate, d.gate_row_stride, d.gate_col_stride = gate.data_ptr(), row, col


class Sampler:
    """The next token of each row of logits from a given uniform number."""

    def __init__(self, vocab):
        self.V = int(vocab)
        self._desc = _lib.SampleDesc(n_tok=0, V=self.V, temperature_all=1.0, top_k_all=0, top_p_all=1.0, min_p_all=0.0)
        check(lib().moe_sample(ctypes.byref(self._desc), None), "moe_sample")       # the size alone: n_tok 0

    def __call__(self, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, probs=None,
                 stream=None):
        """logits [tokens][vocab] f32, bf16 or fp16; u f32 [tokens] in [0, 1) -> tokens int32 [tokens], probs f32
        [tokens] (the share of the kept mass that the token had).

        temperature, top_p, min_p (f32) and top_k (int32): a number for every row, a tensor [tokens], or None
        (temperature 1, nothing cut).  A temperature of 0 takes the largest logit.
        """
        dev = logits.device
        d = _lib.SampleDesc.from_buffer_copy(self._desc)
        d.logits_type = _dtype(logits, "logits")
        d.logits_stride = _rows(logits, self.V, dev, "logits")
        T = logits.shape[0]
        d.logits, d.n_tok = logits.data_ptr(), T
        f32 = torch.float32
        d.u = _vec(u, T, f32, dev, "u")
        if isinstance(temperature, torch.Tensor):
            d.temperature = _vec(temperature, T, f32, dev, "temperature")
        elif temperature is not None:
            d.temperature_all = temperature
        if isinstance(top_k, torch.Tensor):
            d.top_k = _vec(top_k, T, torch.int32, dev, "top_k")
        elif top_k is not None:
            d.top_k_all = top_k
        if isinstance(top_p, torch.Tensor):
            d.top_p = _vec(top_p, T, f32, dev, "top_p")
        elif top_p is not None:
            d.top_p_all = top_p
        if isinstance(min_p, torch.Tensor):
            d.min_p = _vec(min_p, T, f32, dev, "min_p")
        elif min_p is not None:
            d.min_p_all = min_p
        tokens = _out(tokens, (T,), torch.int32, dev, "tokens", stream)
        probs = _out(probs, (T,), f32, dev, "probs", stream)
        d.tokens, d.probs = tokens.data_ptr(), probs.data_ptr()
        ws = _empty((lib().moe_sample_workspace_bytes(T, self.V),), torch.uint8, dev, stream)
        d.workspace = ws.data_ptr()
        _call(lib().moe_sample, d, dev, stream, "moe_sample")
        return tokens, probs
