"""Expert layers and linear maps with 8-bit floating-point weights, over the C ABI.

    fp8_quantize  moe_fp8_quantize: rows to e4m3 and a power of two for each 128 values, or a weight in blocks of 128 x 128
    Fp8Linear     moe_fp8_product: x times a weight [out][in] of e4m3 transposed, a scale for each block of 128 x 128
    Fp8Moe        moe_fp8_layer: a layer of experts with such weights: routing by a ScoredRouter, up and gate, SwiGLU, down
                  and the weighted sum over a token's experts

include/moe_prefetch.h has the formulas.  What block.py says of its objects and calls holds here: an object holds weights and
nothing of a call, a call launches on `stream`, does not synchronise and can be captured into a graph; inference only.
"""
import torch

from . import _lib
from ._lib import lib
from .block import _F32, _I32, DTYPES, _call, _empty, _first, _on_gpu, _out, _place, _rows

_F8 = torch.float8_e4m3fn
BLOCK = 128


def _blocks(n):
    return -(-n // BLOCK)


def _kind(dtype, what):
    d = DTYPES.get(dtype)
    if d is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, not {dtype}")
    return d


def _matrix(t, shape, dtype, dev, what):
    """(row stride, expert stride) of a weight or its scales, [n][k] or [E][n][k] with unit column stride."""
    if t.dtype is not dtype or tuple(t.shape) != shape:
        raise ValueError(f"{what} must be {dtype} {shape}, not {t.dtype} {tuple(t.shape)}")
    if t.get_device() != dev:
        _place(t, dev, what)
    stride = t.stride()
    if shape[-1] > 1 and stride[-1] != 1:
        raise ValueError(f"the columns of {what} must be next to each other, not {stride[-1]} apart")
    ld = stride[-2] if shape[-2] > 1 else shape[-1]
    if ld < shape[-1]:
        raise ValueError(f"the rows of {what} overlap (row stride {ld})")
    ex = stride[0] if len(shape) == 3 and shape[0] > 1 else 0
    return ld, ex


def _weight(q, scale, shape, dev, what):
    """A weight's fields of a descriptor."""
    ld, ex = _matrix(q, shape, _F8, dev, what)
    sld, sex = _matrix(scale, (*shape[:-2], _blocks(shape[-2]), _blocks(shape[-1])), _F32, dev, what + "'s scales")
    return q.data_ptr(), ld, ex, scale.data_ptr(), sld, sex


def _workspace(size, dev, stream):
    """(address, the memory) of a call's workspace"""
    if not size:
        return 0, None
    ws = _empty((size,), torch.uint8, dev, stream)
    return ws.data_ptr(), ws


_quantize = None


def fp8_quantize(x, rows=1, q=None, scale=None, stream=None):
    """x [n][k] f32, bf16 or fp16 -> (q float8_e4m3fn [n][k], scale f32 [n / rows][k / 128], rounded up), x about q times its
    block's scale.  A block has 128 columns and rows rows: 1 (activations) or 128 (weights)."""
    global _quantize
    if _quantize is None:
        _quantize = _lib.packed(_lib.Fp8QuantizeDesc)[0], _lib.entry("moe_fp8_quantize")
    if x.dim() != 2:
        raise ValueError(f"x must be [rows][columns], not {tuple(x.shape)}")
    if rows not in (1, BLOCK):
        raise ValueError(f"blocks have 1 or {BLOCK} rows, not {rows}")
    K = x.shape[1]
    T, ld, dev = _first(x, K, "x")
    kind = _kind(x.dtype, "x")
    s_rows, nb = -(-T // rows), -(-K // BLOCK)
    if q is None:
        q, ldq = _empty((T, K), _F8, dev, stream), K
    elif q.dtype is not _F8:
        raise ValueError(f"q must be {_F8}, not {q.dtype}")
    else:
        ldq = _rows(q, T, K, dev, "q")
    if scale is None:
        scale, lds = _empty((s_rows, nb), _F32, dev, stream), nb
    elif scale.dtype is not _F32:
        raise ValueError(f"scale must be {_F32}, not {scale.dtype}")
    else:
        lds = _rows(scale, s_rows, nb, dev, "scale")
    desc = _quantize[0](x.data_ptr(), ld, kind, rows, T, K, q.data_ptr(), ldq, scale.data_ptr(), lds)
    _call(_quantize[1], desc, dev, stream, "moe_fp8_quantize")
    return q, scale


class Fp8Linear:
    """y = x W^T for W [out][in] of e4m3 codes and scales f32 [out / 128][in / 128], rounded up.  Both are read at each call
    from the memory that they have now."""

    def __init__(self, weight, scale):
        if weight.dim() != 2:
            raise ValueError(f"weight must be [out][in], not {tuple(weight.shape)}")
        self.N, self.K = weight.shape
        self.dev = _on_gpu(weight, "weight")
        self.weight, self.scale = weight.detach(), scale.detach()      # aliases: they keep the memory
        self._w = _weight(weight, scale, (self.N, self.K), self.dev, "weight")
        self._pack, self._fn = _lib.packed(_lib.Fp8ProductDesc)[0], _lib.entry("moe_fp8_product")
        none = self._pack(0, 0, 0, 0, 0, 0, self.N, self.K, *self._w, 0, 0, 0, 0)
        _lib.check(self._fn(none, None), "moe_fp8_product")            # the weight alone: no rows
        self._ws = {}                                                  # rows -> workspace bytes

    def __call__(self, x, x_scale=None, out=None, out_dtype=None, stream=None):
        """x [rows][in] f32, bf16 or fp16, or float8_e4m3fn with x_scale f32 [rows][in / 128] (rounded up) -> y [rows][out] of
        out_dtype: x's, or bf16 for e4m3, unless given."""
        N, K = self.N, self.K
        M, ld, dev = _first(x, K, "x")
        if dev != self.dev:
            raise ValueError(f"the weight is on cuda:{self.dev}, x on cuda:{dev}")
        if x.dtype is _F8:
            if x_scale is None:
                raise ValueError("x of float8_e4m3fn needs x_scale")
            if x_scale.dtype is not _F32:
                raise ValueError(f"x_scale must be {_F32}, not {x_scale.dtype}")
            kind, xs, lds, size = _lib.DTYPE_E4M3, x_scale.data_ptr(), _rows(x_scale, M, _blocks(K), dev, "x_scale"), 0
        else:
            if x_scale is not None:
                raise ValueError(f"x_scale is for x of float8_e4m3fn, not {x.dtype}")
            kind, xs, lds, size = _kind(x.dtype, "x"), 0, 0, self._ws.get(M)
            if size is None:
                size = self._ws[M] = lib().moe_fp8_product_workspace_bytes(M, N, K, kind)
        if out is None:
            if out_dtype is None:
                out_dtype = torch.bfloat16 if x.dtype is _F8 else x.dtype
            to = _kind(out_dtype, "out_dtype")
            out, ldo = _empty((M, N), out_dtype, dev, stream), N
        elif out_dtype is not None and out.dtype is not out_dtype:
            raise ValueError(f"out is {out.dtype}, not {out_dtype}")
        else:
            ldo, to = _rows(out, M, N, dev, "out"), _kind(out.dtype, "out")
        ws, _keep = _workspace(size, dev, stream)
        desc = self._pack(x.data_ptr(), ld, xs, lds, kind, M, N, K, *self._w, out.data_ptr(), ldo, to, ws)
        _call(self._fn, desc, dev, stream, "moe_fp8_product")
        return out


class Fp8Moe:
    """A layer of E experts of e4m3: up and gate [E][intermediate][hidden], down [E][hidden][intermediate], each with scales f32
    [E][rows / 128][columns / 128], rounded up (views of one tensor that holds up and gate are fine).  All are read at each call
    from the memory that they have now.  router: a ScoredRouter over the E experts, for calls that give logits."""

    def __init__(self, up, gate, down, up_scale, gate_scale, down_scale, router=None):
        if up.dim() != 3:
            raise ValueError(f"up must be [experts][intermediate][hidden], not {tuple(up.shape)}")
        self.E, self.I, self.H = E, I, H = tuple(up.shape)
        self.dev = dev = _on_gpu(up, "up")
        if router is not None and router.E != E:
            raise ValueError(f"the router has {router.E} experts, the layer {E}")
        self.router = router
        self.weights = tuple(t.detach() for t in (up, gate, down, up_scale, gate_scale, down_scale))    # aliases
        self._w = (*_weight(gate, gate_scale, (E, I, H), dev, "gate"), *_weight(up, up_scale, (E, I, H), dev, "up"),
                   *_weight(down, down_scale, (E, H, I), dev, "down"))
        self._pack, self._fn = _lib.packed(_lib.Fp8LayerHead)[0], _lib.entry("moe_fp8_layer")
        self._given = bytes(_lib.RouteScoredDesc())
        none = self._pack(0, 0, 0, 0, E, 1, H, I, *self._w, 0, 0, 0, 0, 0, 0)
        _lib.check(self._fn(none + self._given, None), "moe_fp8_layer")         # the weights alone: no tokens
        self._ws = {}                                                           # (tokens, K) -> workspace bytes

    def __call__(self, x, logits=None, ids=None, w=None, out=None, out_dtype=None, stream=None):
        """x [tokens][hidden] f32, bf16 or fp16 -> (out [tokens][hidden] of out_dtype: x's, unless given; ids; w).

        With logits [tokens][E] (f32, bf16 or fp16) the router chooses: ids int32 and w f32 [tokens][K] receive its choice
        (allocated unless given).  Without, ids and w are the choice; an id outside the experts adds nothing.
        """
        E, H = self.E, self.H
        T, ld, dev = _first(x, H, "x")
        if dev != self.dev:
            raise ValueError(f"the weights are on cuda:{self.dev}, x on cuda:{dev}")
        kind = _kind(x.dtype, "x")
        if logits is not None:
            r = self.router
            if r is None:
                raise ValueError("logits need the layer's router")
            K = r.K
            if logits.dim() != 2:
                raise ValueError(f"logits must be [{T}][{E}], not {tuple(logits.shape)}")
            route = r.head(logits, _rows(logits, T, E, dev, "logits"), dev)
            if ids is None:
                ids = _empty((T, K), _I32, dev, stream)
            if w is None:
                w = _empty((T, K), _F32, dev, stream)
        else:
            if ids is None or w is None:
                raise ValueError("either logits, or ids and w")
            if ids.dim() != 2:
                raise ValueError(f"ids must be [{T}][experts of a token], not {tuple(ids.shape)}")
            K, route = ids.shape[1], self._given
        pair = (T, K)
        if out is None:
            out_dtype = x.dtype if out_dtype is None else out_dtype
            to = _kind(out_dtype, "out_dtype")
            out, ldo = _empty((T, H), out_dtype, dev, stream), H
        elif out_dtype is not None and out.dtype is not out_dtype:
            raise ValueError(f"out is {out.dtype}, not {out_dtype}")
        else:
            ldo, to = _rows(out, T, H, dev, "out"), _kind(out.dtype, "out")
        size = self._ws.get(pair)
        if size is None:
            size = self._ws[pair] = lib().moe_fp8_layer_workspace_bytes(T, E, K, H, self.I)
        ws, _keep = _workspace(size, dev, stream)
        desc = self._pack(x.data_ptr(), ld, kind, T, E, K, H, self.I, *self._w, _out(ids, pair, _I32, dev, "ids"),
                          _out(w, pair, _F32, dev, "w"), out.data_ptr(), ldo, to, ws)
        _call(self._fn, desc + route, dev, stream, "moe_fp8_layer")
        return out, ids, w
