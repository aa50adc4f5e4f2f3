"""Temporal operators on the GPU, beside the network's ConvGRU: the other two ways of carrying a stream's past.

The reference's only memory of a stream is the ConvGRU state (model/decoder.py:152-190): these have no
counterpart there.  They keep its contract (model/decoder.py:174-180): the caller owns the state, and one call with T steps gives
what T calls with one step give.

* a state of fixed size: ``causal_conv`` (a short depthwise filter over time) and ``selective_scan`` (a state space scan with
  step sizes and projections that depend on the input);
* a memory that grows: ``append_kv`` stores a stream's tokens in a paged key-value cache, rotated by their position, and
  ``attend`` reads it - for one new token per stream or for whole chunks of different lengths.

Everything is channels-last.  Tensors are fp32, fp16 or bf16 on one HIP device; sums, states and softmax statistics are
fp32.  Work goes to the current stream of the tensors' device, nothing synchronises, every call can be captured into a HIP
graph.  Inference only, like the network: tensors that need a gradient or carry a tangent are refused.  No CPU fallback.
"""
import functools
import struct

import torch
from torch.autograd import forward_ad as _forward

from . import native

_DTYPES = {torch.float32: native.DTYPE_F32, torch.float16: native.DTYPE_F16, torch.bfloat16: native.DTYPE_BF16IO}
_F32, _I32 = torch.float32, torch.int32
_grad, _empty_like = torch.is_grad_enabled, torch.empty_like
_stream_of, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


# ---- arguments.  A call with a single step per stream is bound by the host, so each operator checks its arguments in one
# expression; only a call that fails it comes here, to be told what is wrong
def _tensor(what, t, dtype, dev, shape):
    """One tensor argument: type, device and shape (-1: any size), and no gradient."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError("%s must be a tensor" % what)
    if t.device != dev:
        raise RuntimeError("%s must be on %s, not on %s" % (what, dev, t.device))
    if t.dtype != dtype:
        raise RuntimeError("%s must be %s, not %s" % (what, dtype, t.dtype))
    if len(t.shape) != len(shape) or any(b >= 0 and a != b for a, b in zip(t.shape, shape)):
        raise RuntimeError("%s has shape %s, expected %s" % (what, tuple(t.shape), tuple("any" if b < 0 else b for b in shape)))
    if t.requires_grad and _grad():
        raise RuntimeError("%s needs a gradient: the temporal operators are inference only" % what)
    if _forward._current_level >= 0 and _dual(t):
        raise RuntimeError("%s carries a tangent: the temporal operators are inference only" % what)


def _dual(*tensors):
    """Whether one of them carries a tangent.  (To be asked inside a dual level only; no_grad does not end forward mode.)"""
    return torch._C._is_fwd_grad_enabled() and any(t is not None and _forward.unpack_dual(t).tangent is not None for t in tensors)


def _lead(what, t):
    """The three-dimensional tensor that the others are checked against."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise RuntimeError("%s must be a HIP device tensor (no CPU fallback)" % what)
    if t.dtype not in _DTYPES:
        raise RuntimeError("%s: unsupported dtype %s (float32 / float16 / bfloat16)" % (what, t.dtype))
    _tensor(what, t, t.dtype, t.device, (-1, -1, -1))
    return t.device, t.dtype, t.shape


def _refuse_conv(x, weight, bias, state):
    dev, dt, (B, T, D) = _lead("x", x)
    _tensor("weight", weight, dt, dev, (-1, D))
    W = weight.shape[0]
    if not 2 <= W <= 4:
        raise RuntimeError("weight: the filter has 2 to 4 taps, not %d" % W)
    if bias is not None:
        _tensor("bias", bias, dt, dev, (D,))
    if state is not None:
        _tensor("state", state, dt, dev, (B, W - 1, D))
    raise RuntimeError("causal_conv: bad arguments")


def _refuse_scan(x, dt, A, B, C, D, z, dt_bias, state):
    dev, ty, (nb, T, nd) = _lead("x", x)
    _tensor("dt", dt, ty, dev, (nb, T, nd))
    _tensor("A", A, _F32, dev, (-1, nd))
    N = A.shape[0]
    if not 1 <= N <= 64:
        raise RuntimeError("A: 1 to 64 states per channel, not %d" % N)
    _tensor("B", B, ty, dev, (nb, T, N))
    _tensor("C", C, ty, dev, (nb, T, N))
    for what, t, kind, shape in (("z", z, ty, (nb, T, nd)), ("D", D, _F32, (nd,)), ("dt_bias", dt_bias, _F32, (nd,)), ("state", state, _F32, (nb, N, nd))):
        if t is not None:
            _tensor(what, t, kind, dev, shape)
    raise RuntimeError("selective_scan: bad arguments")


def _refuse_paged(what, rows, cache, table, lengths, offsets):
    dev, dt, (M, H, Dh) = _lead(what, rows)
    if not (isinstance(cache, (tuple, list)) and len(cache) == 2):
        raise RuntimeError("cache must be the pair (key pages, value pages)")
    kp, vp = cache
    _tensor("key pages", kp, dt, dev, (-1, -1, -1, Dh))
    _tensor("value pages", vp, dt, dev, kp.shape)
    if not (kp.is_contiguous() and vp.is_contiguous()):
        raise RuntimeError("the pages must be dense")
    _tensor("table", table, _I32, dev, (-1, -1))
    S = table.shape[0]
    _tensor("lengths", lengths, _I32, dev, (S,))
    if offsets is not None:
        _tensor("offsets", offsets, _I32, dev, (S + 1,))
    if not (table.is_contiguous() and lengths.is_contiguous() and (offsets is None or offsets.is_contiguous())):
        raise RuntimeError("table, lengths and offsets must be dense")
    if offsets is None and M != S:
        raise RuntimeError("without offsets every stream has one row: %d rows for %d streams" % (M, S))
    if M and not S:
        raise RuntimeError("%d rows for no stream" % M)


def _refuse_append(k, v, cache, table, lengths, offsets, freqs, q):
    _refuse_paged("k", k, cache, table, lengths, offsets)
    dev, dt, (M, H, Dh) = _lead("k", k)
    _tensor("v", v, dt, dev, (M, H, Dh))
    if H != cache[0].shape[1]:
        raise RuntimeError("k has %d heads, the pages have %d" % (H, cache[0].shape[1]))
    if freqs is not None:
        _tensor("freqs", freqs, _F32, dev, (-1,))
    if q is not None:
        _tensor("q", q, dt, dev, (M, -1, Dh))
    raise RuntimeError("append_kv: bad arguments")


def _fits(rows, dt, di, kp, vp, table, lengths, offsets):
    """Whether what append_kv and attend share is as it should be."""
    M, _, Dh = rows.shape
    S, _ = table.shape
    P, Hkv, page, _ = shape = kp.shape
    return (rows.is_cuda and shape == (P, Hkv, page, Dh) and vp.shape == shape and kp.dtype is dt and vp.dtype is dt and kp.get_device() == di and
            vp.get_device() == di and kp.is_contiguous() and vp.is_contiguous() and table.dtype is _I32 and lengths.dtype is _I32 and
            lengths.shape == (S,) and table.get_device() == di and lengths.get_device() == di and table.is_contiguous() and
            lengths.is_contiguous() and (S or not M) and
            (M == S if offsets is None else offsets.dtype is _I32 and offsets.shape == (S + 1,) and offsets.get_device() == di and offsets.is_contiguous()) and
            not ((rows.requires_grad or kp.requires_grad or vp.requires_grad) and _grad()) and
            not (_forward._current_level >= 0 and _dual(rows, kp, vp)))


def _dense_last(t):
    """The tensor, or a dense copy where its channels are not next to each other."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _rows(t, per):
    """[rows, heads, dim] in 16-byte pieces (``per`` elements) - as it is, or a dense copy - its address and its two strides."""
    s0, s1, s2 = t.stride()
    at = t.data_ptr()
    if s2 == 1 and not (s0 % per or s1 % per or at % 16):
        return t, at, s0, s1
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), t.stride(0), t.stride(1)


def _dense_like(t):
    """A new dense tensor of t's shape and type (``empty_like`` of a dense one: a quarter less of the host's time)."""
    return _empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _call(entry, code, block, index):
    """One native call on the tensors' device and its current stream."""
    if _current_device() == index:
        rc = entry(code, block, _stream_of(index))
    else:
        with torch.cuda.device(index):
            rc = entry(code, block, _stream_of(index))
    if rc:
        native.check(rc, entry.__name__)


_CONV = struct.Struct("6P7q")


def causal_conv(x, weight, bias=None, state=None, silu=True):
    """Depthwise filter over the last W steps: ``y[b,t,d] = act(bias[d] + sum_w weight[w,d] xx[b,t+w,d])`` with ``xx`` the
    ``W-1`` rows of ``state`` (None: zeros) followed by ``x``; ``act`` is silu or nothing.

    ``x`` [B,T,D] (any strides between rows, e.g. a slice of a projection), ``weight`` [W,D] with W = 2..4, ``bias`` [D],
    ``state`` [B,W-1,D], all of one dtype.  Returns ``(y, new state)``; the new state is the last W-1 rows of ``xx``."""
    try:
        dt, di, (B, T, D), W = x.dtype, x.get_device(), x.shape, weight.shape[0]
        ok = (x.is_cuda and dt in _DTYPES and weight.dtype is dt and weight.shape == (W, D) and weight.get_device() == di and 2 <= W <= 4 and
              (bias is None or (bias.dtype is dt and bias.shape == (D,) and bias.get_device() == di)) and
              (state is None or (state.dtype is dt and state.shape == (B, W - 1, D) and state.get_device() == di)) and
              not (_grad() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                (state is not None and state.requires_grad))) and
              not (_forward._current_level >= 0 and _dual(x, weight, bias, state)))
    except (AttributeError, ValueError, IndexError):
        ok = False
    if not ok:
        _refuse_conv(x, weight, bias, state)
    x, weight = _dense_last(x), weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if state is None:
        new = x.new_empty((B, W - 1, D))
    else:
        state = state.contiguous()
        new = _empty_like(state)
    y = _dense_like(x)
    sb, st, _ = x.stride()
    _call(native.lib().rvm_causal_conv, _DTYPES[dt],
          _CONV.pack(x.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), 0 if state is None else state.data_ptr(),
                     y.data_ptr(), new.data_ptr(), sb, st, B, T, D, W, bool(silu)), di)
    return y, new


_SCAN = struct.Struct("12P16q")


@functools.lru_cache(maxsize=1024)
def _scan_workspace(B, T, D, N):
    """Bytes, by the sizes alone."""
    need = native.lib().rvm_selective_scan_workspace(B, T, D, N)
    if need < 0:
        raise RuntimeError("selective_scan: bad shape")
    return need


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, softplus=True):
    """Selective state space scan: ``delta = softplus(dt + dt_bias)``, ``h_t = exp(delta_t A) h_(t-1) + delta_t x_t B_t``,
    ``y_t = sum_n C_t[n] h_t[n] + D x_t``, times ``z_t sigmoid(z_t)`` where ``z`` is given.

    ``x``, ``dt``, ``z`` [b,T,d] and ``B``, ``C`` [b,T,N] of one dtype (any strides between rows), N = 1..64; ``A`` [N,d],
    ``D`` [d], ``dt_bias`` [d] and ``state`` [b,N,d] (None: zeros) in fp32.  Returns ``(y, new state)``.  Without ``softplus``
    the step size is ``dt + dt_bias`` itself."""
    try:
        ty, di, xs, N = x.dtype, x.get_device(), x.shape, A.shape[0]
        nb, T, nd = xs
        bc = (nb, T, N)
        ok = (x.is_cuda and ty in _DTYPES and dt.dtype is ty and dt.shape == xs and dt.get_device() == di and
              A.dtype is _F32 and A.shape == (N, nd) and A.get_device() == di and 1 <= N <= 64 and
              B.dtype is ty and B.shape == bc and B.get_device() == di and C.dtype is ty and C.shape == bc and C.get_device() == di and
              (D is None or (D.dtype is _F32 and D.shape == (nd,) and D.get_device() == di)) and
              (z is None or (z.dtype is ty and z.shape == xs and z.get_device() == di)) and
              (dt_bias is None or (dt_bias.dtype is _F32 and dt_bias.shape == (nd,) and dt_bias.get_device() == di)) and
              (state is None or (state.dtype is _F32 and state.shape == (nb, N, nd) and state.get_device() == di)) and
              not (_grad() and any(t is not None and t.requires_grad for t in (x, dt, A, B, C, D, z, dt_bias, state))) and
              not (_forward._current_level >= 0 and _dual(x, dt, A, B, C, D, z, dt_bias, state)))
    except (AttributeError, ValueError, IndexError):
        ok = False
    if not ok:
        _refuse_scan(x, dt, A, B, C, D, z, dt_bias, state)
    x, dt, B, C, A = _dense_last(x), _dense_last(dt), _dense_last(B), _dense_last(C), A.contiguous()
    zp = z_sb = z_st = 0
    if z is not None:
        z = _dense_last(z)
        zp, (z_sb, z_st, _) = z.data_ptr(), z.stride()
    if D is not None:
        D = D.contiguous()
    if dt_bias is not None:
        dt_bias = dt_bias.contiguous()
    if state is None:
        new = A.new_empty((nb, N, nd))
    else:
        state = state.contiguous()
        new = _empty_like(state)
    y = _dense_like(x)
    need = _scan_workspace(nb, T, nd, N)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    xs, ds, Bs, Cs = x.stride(), dt.stride(), B.stride(), C.stride()
    _call(native.lib().rvm_selective_scan, _DTYPES[ty],
          _SCAN.pack(x.data_ptr(), dt.data_ptr(), zp, B.data_ptr(), C.data_ptr(), A.data_ptr(), 0 if D is None else D.data_ptr(),
                     0 if dt_bias is None else dt_bias.data_ptr(), 0 if state is None else state.data_ptr(), y.data_ptr(), new.data_ptr(),
                     ws.data_ptr() if need else 0, xs[0], xs[1], ds[0], ds[1], z_sb, z_st, Bs[0], Bs[1], Cs[0], Cs[1],
                     nb, T, nd, N, bool(softplus), need), di)
    return y, new


_APPEND = struct.Struct("10P16q")


def append_kv(k, v, cache, table, lengths, offsets=None, freqs=None, q=None, interleaved=False):
    """Stores new tokens in a paged cache, in place, the keys rotated by their position; with ``q`` also returns the queries
    rotated the same way (the new tensor that ``attend`` takes), else None.

    ``cache`` = (key pages, value pages), each dense [pages, kv heads, page, dim]; position p of stream s lives in page
    ``table[s, p // page]``, slot ``p % page``.  ``k``, ``v`` [M, kv heads, dim] and ``q`` [M, heads, dim] are the new tokens'
    rows, stream after stream: stream s has the rows ``offsets[s] .. offsets[s+1]`` (None: one row per stream), and its i-th
    row gets position ``lengths[s] + i`` - ``lengths`` counts the tokens BEFORE this call.  ``table`` [S, columns],
    ``lengths`` [S] and ``offsets`` [S+1] are int32 on the device.  A negative position is no token and stores nothing; a
    token whose page is not in the pool, or not in the table, is dropped.  Two rows must not share a slot.

    ``freqs`` (fp32, radians per position; None: no rotation) turns the first ``2 * len(freqs)`` dims, a multiple of 16: the
    pairs (i, i + len(freqs)), or (2i, 2i+1) with ``interleaved``."""
    try:
        kp, vp = cache
        dt, di, ks, qs = k.dtype, k.get_device(), k.shape, k.shape if q is None else q.shape
        M, H, Dh = ks
        ok = (dt in _DTYPES and _fits(k, dt, di, kp, vp, table, lengths, offsets) and kp.shape[1] == H and v.dtype is dt and v.shape == ks and
              v.get_device() == di and (q is None or (q.dtype is dt and qs == (M, qs[1], Dh) and q.get_device() == di)) and
              (freqs is None or (freqs.dtype is _F32 and freqs.dim() == 1 and freqs.get_device() == di)) and
              not (_grad() and (v.requires_grad or (q is not None and q.requires_grad) or (freqs is not None and freqs.requires_grad))) and
              not (_forward._current_level >= 0 and _dual(v, q, freqs)))
    except (AttributeError, ValueError, IndexError, TypeError):
        ok = False
    if not ok:
        _refuse_append(k, v, cache, table, lengths, offsets, freqs, q)
    per = 4 if dt is _F32 else 8
    k, k_at, k_sm, k_sh = _rows(k, per)
    v, v_at, v_sm, v_sh = _rows(v, per)
    rot = fp = q_at = out_at = q_sm = q_sh = 0
    out = None
    if freqs is not None:
        freqs = freqs.contiguous()
        rot, fp = 2 * freqs.shape[0], freqs.data_ptr()
    if q is not None:
        q, q_at, q_sm, q_sh = _rows(q, per)
        out = _dense_like(q)
        out_at = out.data_ptr()
    S, width = table.shape
    _call(native.lib().rvm_append_kv, _DTYPES[dt],
          _APPEND.pack(q_at, k_at, v_at, out_at, kp.data_ptr(), vp.data_ptr(), table.data_ptr(), lengths.data_ptr(),
                       0 if offsets is None else offsets.data_ptr(), fp, q_sm, q_sh, k_sm, k_sh, v_sm, v_sh,
                       M, S, qs[1], H, Dh, kp.shape[0], kp.shape[2], width, rot, bool(interleaved)), di)
    return out


_ATTEND = struct.Struct("8P11qd")


@functools.lru_cache(maxsize=1024)
def _attend_workspace(code, packed, *sizes):
    """Bytes, by the sizes alone (``packed``: whether the rows come with offsets)."""
    need = native.lib().rvm_attend_workspace(code, _ATTEND.pack(0, 0, 0, 0, 0, 16, 16, 16 * packed, 0, 0, *sizes, 0, 1.0))
    if need < 0:
        native.check(1, "rvm_attend_workspace")
    return need


def attend(q, cache, table, lengths, offsets=None, scale=None):
    """Attention of new tokens over their streams' caches: ``softmax_j(scale q . k_j) v_j`` over the positions up to the row's
    own, ``lengths[s] + i`` (the rows' own keys are appended first, with the same arguments).  ``q`` [M, heads, dim]; query
    head h reads key head ``h // (heads / kv heads)``; ``scale`` defaults to ``dim ** -0.5``.  Returns [M, heads, dim].

    ``scale`` must be positive and finite in fp32.  Rows of more than 32 streams (with ``offsets``) are not cut along their keys: where
    a few of many streams have much longer memories, calls of up to 32 streams are faster.

    A row with a negative position, or behind the last stream's rows, gives 0.  Pages outside the pool are not followed:
    a row that would read one gives NaN."""
    try:
        kp, vp = cache
        dt, di = q.dtype, q.get_device()
        ok = dt in _DTYPES and _fits(q, dt, di, kp, vp, table, lengths, offsets)
    except (AttributeError, ValueError, IndexError, TypeError):
        ok = False
    if not ok:
        _refuse_paged("q", q, cache, table, lengths, offsets)
        raise RuntimeError("attend: bad arguments")
    M, Hq, Dh = q.shape
    P, Hkv, page, _ = kp.shape
    S, width = table.shape
    code = _DTYPES[dt]
    need = _attend_workspace(code, offsets is not None, M, S, Hq, Hkv, Dh, P, page, width)
    q, q_at, sm, sh = _rows(q, 4 if dt is _F32 else 8)
    out = _dense_like(q)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _call(native.lib().rvm_attend, code,
          _ATTEND.pack(q_at, kp.data_ptr(), vp.data_ptr(), out.data_ptr(), ws.data_ptr() if need else 0, table.data_ptr(),
                       lengths.data_ptr(), 0 if offsets is None else offsets.data_ptr(), sm, sh, M, S, Hq, Hkv, Dh, P, page, width, need,
                       Dh ** -0.5 if scale is None else float(scale)), di)
    return out
