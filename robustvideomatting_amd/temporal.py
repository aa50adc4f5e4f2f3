"""Temporal operators on the GPU, beside the network's ConvGRU: the other two ways of carrying a stream's past.

The reference's only memory of a stream is the ConvGRU state (/root/reference/model/decoder.py:152-190): these have no
counterpart there.  They keep its contract (decoder.py:174-180): the caller owns the state, and one call with T steps gives
what T calls with one step give.

* a state of fixed size: ``causal_conv`` (a short depthwise filter over time) and ``selective_scan`` (a state space scan with
  step sizes and projections that depend on the input);
* a memory that grows: ``append_kv`` stores a stream's tokens in a paged key-value cache, rotated by their position, and
  ``attend`` reads it - for one new token per stream or for whole chunks of different lengths.

Everything is channels-last.  Tensors are fp32, fp16 or bf16 on one HIP device; sums, states and softmax statistics are
fp32.  Work goes to the current stream of the tensors' device, nothing synchronises, every call can be captured into a HIP
graph.  Inference only, like the network: tensors that need a gradient are refused.  No CPU fallback.
"""
import struct

import torch

from . import native

_DTYPES = {torch.float32: native.DTYPE_F32, torch.float16: native.DTYPE_F16, torch.bfloat16: native.DTYPE_BF16IO}


def _refuse(what, t, dtype, dev, shape):
    """Says what is wrong with a tensor argument (-1 in shape: any size)."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError("%s must be a tensor" % what)
    if t.device != dev:
        raise RuntimeError("%s must be on %s, not on %s" % (what, dev, t.device))
    if t.dtype != dtype:
        raise RuntimeError("%s must be %s, not %s" % (what, dtype, t.dtype))
    if len(t.shape) != len(shape) or any(b >= 0 and a != b for a, b in zip(t.shape, shape)):
        raise RuntimeError("%s has shape %s, expected %s" % (what, tuple(t.shape), tuple("any" if b < 0 else b for b in shape)))
    raise RuntimeError("%s needs a gradient: the temporal operators are inference only" % what)


def _need(what, t, dtype, dev, shape):
    """One tensor argument: type, device and shape, and no gradient.  (Single steps are bound by the host: this is their path.)"""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == dev.index) or \
            (t.requires_grad and torch.is_grad_enabled()):
        _refuse(what, t, dtype, dev, shape)


def _lead(what, t, ndim):
    """The tensor that the others are checked against: -> (dtype code, device, dtype, shape)."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise RuntimeError("%s must be a HIP device tensor (no CPU fallback)" % what)
    dtype, dev, shape = t.dtype, t.device, t.shape
    code = _DTYPES.get(dtype)
    if code is None:
        raise RuntimeError("%s: unsupported dtype %s (float32 / float16 / bfloat16)" % (what, dtype))
    if len(shape) != ndim or (t.requires_grad and torch.is_grad_enabled()):
        _refuse(what, t, dtype, dev, (-1,) * ndim)
    return code, dev, dtype, shape


def _dense_last(t):
    """The tensor, or a dense copy where its channels are not next to each other."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _rows(t):
    """[rows, heads, dim] in 16-byte pieces: as it is, or a dense copy."""
    s0, s1, s2 = t.stride()
    per = 16 // t.element_size()
    return t if s2 == 1 and s0 % per == 0 and s1 % per == 0 and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


_stream_of, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _call(entry, code, block, dev):
    """One native call on the tensors' device and its current stream."""
    index = dev.index
    if _current_device() == index:
        rc = entry(code, block, _stream_of(index))
    else:
        with torch.cuda.device(dev):
            rc = entry(code, block, _stream_of(index))
    if rc:
        native.check(rc, entry.__name__)


_CONV = struct.Struct("6P7q")


def causal_conv(x, weight, bias=None, state=None, silu=True):
    """Depthwise filter over the last W steps: ``y[b,t,d] = act(bias[d] + sum_w weight[w,d] xx[b,t+w,d])`` with ``xx`` the
    ``W-1`` rows of ``state`` (None: zeros) followed by ``x``; ``act`` is silu or nothing.

    ``x`` [B,T,D] (any strides between rows, e.g. a slice of a projection), ``weight`` [W,D] with W = 2..4, ``bias`` [D],
    ``state`` [B,W-1,D], all of one dtype.  Returns ``(y, new state)``; the new state is the last W-1 rows of ``xx``."""
    code, dev, dt, (B, T, D) = _lead("x", x, 3)
    W = len(weight) if isinstance(weight, torch.Tensor) and weight.ndim else -1
    _need("weight", weight, dt, dev, (W, D))
    if not 2 <= W <= 4:
        raise RuntimeError("weight: the filter has 2 to 4 taps, not %d" % W)
    x, weight = _dense_last(x), weight.contiguous()
    bp = sp = 0
    if bias is not None:
        _need("bias", bias, dt, dev, (D,))
        bias = bias.contiguous()
        bp = bias.data_ptr()
    if state is not None:
        _need("state", state, dt, dev, (B, W - 1, D))
        state = state.contiguous()
        sp = state.data_ptr()
    y, new = x.new_empty((B, T, D)), x.new_empty((B, W - 1, D))
    sb, st, _ = x.stride()
    _call(native.lib().rvm_causal_conv, code,
          _CONV.pack(x.data_ptr(), weight.data_ptr(), bp, sp, y.data_ptr(), new.data_ptr(), sb, st, B, T, D, W, bool(silu)), dev)
    return y, new


_SCAN = struct.Struct("12P16q")


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, softplus=True):
    """Selective state space scan: ``delta = softplus(dt + dt_bias)``, ``h_t = exp(delta_t A) h_(t-1) + delta_t x_t B_t``,
    ``y_t = sum_n C_t[n] h_t[n] + D x_t``, times ``z_t sigmoid(z_t)`` where ``z`` is given.

    ``x``, ``dt``, ``z`` [b,T,d] and ``B``, ``C`` [b,T,N] of one dtype (any strides between rows), N = 1..64; ``A`` [N,d],
    ``D`` [d], ``dt_bias`` [d] and ``state`` [b,N,d] (None: zeros) in fp32.  Returns ``(y, new state)``.  Without ``softplus``
    the step size is ``dt + dt_bias`` itself."""
    code, dev, ty, (nb, T, nd) = _lead("x", x, 3)
    f32 = torch.float32
    _need("dt", dt, ty, dev, (nb, T, nd))
    N = len(A) if isinstance(A, torch.Tensor) and A.ndim else -1
    _need("A", A, f32, dev, (N, nd))
    if not 1 <= N <= 64:
        raise RuntimeError("A: 1 to 64 states per channel, not %d" % N)
    _need("B", B, ty, dev, (nb, T, N))
    _need("C", C, ty, dev, (nb, T, N))
    x, dt, B, C, A = _dense_last(x), _dense_last(dt), _dense_last(B), _dense_last(C), A.contiguous()
    zp = z_sb = z_st = 0
    if z is not None:
        _need("z", z, ty, dev, (nb, T, nd))
        z = _dense_last(z)
        zp, (z_sb, z_st, _) = z.data_ptr(), z.stride()
    Dp = bp = hp = 0
    if D is not None:
        _need("D", D, f32, dev, (nd,))
        D = D.contiguous()
        Dp = D.data_ptr()
    if dt_bias is not None:
        _need("dt_bias", dt_bias, f32, dev, (nd,))
        dt_bias = dt_bias.contiguous()
        bp = dt_bias.data_ptr()
    if state is not None:
        _need("state", state, f32, dev, (nb, N, nd))
        state = state.contiguous()
        hp = state.data_ptr()
    y, new = x.new_empty((nb, T, nd)), A.new_empty((nb, N, nd))
    L = native.lib()
    need = L.rvm_selective_scan_workspace(nb, T, nd, N)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    xs, ds, Bs, Cs = x.stride(), dt.stride(), B.stride(), C.stride()
    _call(L.rvm_selective_scan, code,
          _SCAN.pack(x.data_ptr(), dt.data_ptr(), zp, B.data_ptr(), C.data_ptr(), A.data_ptr(), Dp, bp, hp, y.data_ptr(), new.data_ptr(),
                     ws.data_ptr() if ws is not None else 0, xs[0], xs[1], ds[0], ds[1], z_sb, z_st, Bs[0], Bs[1], Cs[0], Cs[1],
                     nb, T, nd, N, bool(softplus), need), dev)
    return y, new


def _paged(what, rows, cache, table, lengths, offsets):
    """Checks of what append_kv and attend share; ``rows`` is the tensor of the new rows."""
    code, dev, dt, (M, H, Dh) = _lead(what, rows, 3)
    if not (isinstance(cache, (tuple, list)) and len(cache) == 2):
        raise RuntimeError("cache must be the pair (key pages, value pages)")
    kp, vp = cache
    P, Hkv, page, _ = kp.shape if isinstance(kp, torch.Tensor) and kp.ndim == 4 else (-1, -1, -1, -1)
    _need("key pages", kp, dt, dev, (P, Hkv, page, Dh))
    _need("value pages", vp, dt, dev, (P, Hkv, page, Dh))
    if not (kp.is_contiguous() and vp.is_contiguous()):
        raise RuntimeError("the pages must be dense")
    S, width = table.shape if isinstance(table, torch.Tensor) and table.ndim == 2 else (-1, -1)
    _need("table", table, torch.int32, dev, (S, width))
    _need("lengths", lengths, torch.int32, dev, (S,))
    if not (table.is_contiguous() and lengths.is_contiguous()):
        raise RuntimeError("table and lengths must be dense")
    op = 0
    if offsets is not None:
        _need("offsets", offsets, torch.int32, dev, (S + 1,))
        if not offsets.is_contiguous():
            raise RuntimeError("offsets must be dense")
        op = offsets.data_ptr()
    elif M != S:
        raise RuntimeError("without offsets every stream has one row: %d rows for %d streams" % (M, S))
    if M and not S:
        raise RuntimeError("%d rows for no stream" % M)
    return code, dev, dt, kp, vp, (M, S, H, Hkv, Dh, P, page, width), (table.data_ptr(), lengths.data_ptr(), op)


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
    code, dev, dt, kp, vp, (M, S, H, Hkv, Dh, P, page, width), meta = _paged("k", k, cache, table, lengths, offsets)
    _need("v", v, dt, dev, (M, H, Dh))
    if H != Hkv:
        raise RuntimeError("k has %d heads, the pages have %d" % (H, Hkv))
    k, v = _rows(k), _rows(v)
    rot = fp = qp = out_p = q_sm = q_sh = 0
    Hq, out = Hkv, None
    if freqs is not None:
        n = freqs.numel() if isinstance(freqs, torch.Tensor) else -1
        _need("freqs", freqs, torch.float32, dev, (n,))
        freqs = freqs.contiguous()
        rot, fp = 2 * n, freqs.data_ptr()
    if q is not None:
        Hq = q.shape[1] if isinstance(q, torch.Tensor) and q.ndim == 3 else -1
        _need("q", q, dt, dev, (M, Hq, Dh))
        q = _rows(q)
        out = k.new_empty((M, Hq, Dh))
        qp, out_p, (q_sm, q_sh, _) = q.data_ptr(), out.data_ptr(), q.stride()
    k_sm, k_sh, _ = k.stride()
    v_sm, v_sh, _ = v.stride()
    _call(native.lib().rvm_append_kv, code,
          _APPEND.pack(qp, k.data_ptr(), v.data_ptr(), out_p, kp.data_ptr(), vp.data_ptr(), *meta, fp, q_sm, q_sh, k_sm, k_sh, v_sm, v_sh,
                       M, S, Hq, Hkv, Dh, P, page, width, rot, bool(interleaved)), dev)
    return out


_ATTEND = struct.Struct("8P11qd")


def attend(q, cache, table, lengths, offsets=None, scale=None):
    """Attention of new tokens over their streams' caches: ``softmax_j(scale q . k_j) v_j`` over the positions up to the row's
    own, ``lengths[s] + i`` (the rows' own keys are appended first, with the same arguments).  ``q`` [M, heads, dim]; query
    head h reads key head ``h // (heads / kv heads)``; ``scale`` defaults to ``dim ** -0.5``.  Returns [M, heads, dim].

    A row with a negative position, or behind the last stream's rows, gives 0.  Pages outside the pool are not followed:
    a row that would read one gives NaN."""
    code, dev, dt, kp, vp, sizes, meta = _paged("q", q, cache, table, lengths, offsets)
    M, S, Hq, Hkv, Dh, P, page, width = sizes
    q = _rows(q)
    out = q.new_empty((M, Hq, Dh))
    L = native.lib()
    scale = Dh ** -0.5 if scale is None else float(scale)
    sm, sh, _ = q.stride()
    head = (q.data_ptr(), kp.data_ptr(), vp.data_ptr(), out.data_ptr())
    need = L.rvm_attend_workspace(code, _ATTEND.pack(*head, 0, *meta, sm, sh, *sizes, 0, scale))
    if need < 0:
        native.check(1, "rvm_attend_workspace")
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(L.rvm_attend, code, _ATTEND.pack(*head, ws.data_ptr() if need else 0, *meta, sm, sh, *sizes, need, scale), dev)
    return out
