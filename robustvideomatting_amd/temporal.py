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


def _check(what, t, dtype, dev, shape):
    """One tensor argument: type, device and shape (-1: any size)."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError("%s must be a tensor" % what)
    if t.device != dev:
        raise RuntimeError("%s must be on %s, not on %s" % (what, dev, t.device))
    if t.dtype != dtype:
        raise RuntimeError("%s must be %s, not %s" % (what, dtype, t.dtype))
    if len(t.shape) != len(shape) or any(b >= 0 and a != b for a, b in zip(t.shape, shape)):
        raise RuntimeError("%s has shape %s, expected %s" % (what, tuple(t.shape), tuple("any" if b < 0 else b for b in shape)))
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("%s needs a gradient: the temporal operators are inference only" % what)


def _first(what, t):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise RuntimeError("%s must be a HIP device tensor (no CPU fallback)" % what)
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise RuntimeError("%s: unsupported dtype %s (float32 / float16 / bfloat16)" % (what, t.dtype))
    return code


def _dense_last(t):
    """The tensor, or a dense copy where its channels are not next to each other."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _rows(t):
    """[rows, heads, dim] in 16-byte pieces: as it is, or a dense copy."""
    s0, s1, s2 = t.stride()
    per = 16 // t.element_size()
    return t if s2 == 1 and s0 % per == 0 and s1 % per == 0 and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _call(entry, code, block, dev):
    """One native call on the tensors' device and its current stream."""
    stream = torch._C._cuda_getCurrentRawStream(dev.index)
    if torch._C._cuda_getDevice() == dev.index:
        rc = entry(code, block, stream)
    else:
        with torch.cuda.device(dev):
            rc = entry(code, block, stream)
    if rc:
        native.check(rc, entry.__name__)


_CONV = struct.Struct("6P7q")


def causal_conv(x, weight, bias=None, state=None, silu=True):
    """Depthwise filter over the last W steps: ``y[b,t,d] = act(bias[d] + sum_w weight[w,d] xx[b,t+w,d])`` with ``xx`` the
    ``W-1`` rows of ``state`` (None: zeros) followed by ``x``; ``act`` is silu or nothing.

    ``x`` [B,T,D] (any strides between rows, e.g. a slice of a projection), ``weight`` [W,D] with W = 2..4, ``bias`` [D],
    ``state`` [B,W-1,D], all of one dtype.  Returns ``(y, new state)``; the new state is the last W-1 rows of ``xx``."""
    code = _first("x", x)
    dev, dt = x.device, x.dtype
    _check("x", x, dt, dev, (-1, -1, -1))
    B, T, D = x.shape
    _check("weight", weight, dt, dev, (-1, D))
    W = weight.shape[0]
    if not 2 <= W <= 4:
        raise RuntimeError("weight: the filter has 2 to 4 taps, not %d" % W)
    x, weight = _dense_last(x), weight.contiguous()
    bp = sp = 0
    if bias is not None:
        _check("bias", bias, dt, dev, (D,))
        bias = bias.contiguous()
        bp = bias.data_ptr()
    if state is not None:
        _check("state", state, dt, dev, (B, W - 1, D))
        state = state.contiguous()
        sp = state.data_ptr()
    y = torch.empty((B, T, D), dtype=dt, device=dev)
    new = torch.empty((B, W - 1, D), dtype=dt, device=dev)
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
    code = _first("x", x)
    dev, ty, f32 = x.device, x.dtype, torch.float32
    _check("x", x, ty, dev, (-1, -1, -1))
    nb, T, nd = x.shape
    _check("dt", dt, ty, dev, (nb, T, nd))
    _check("A", A, f32, dev, (-1, nd))
    N = A.shape[0]
    if not 1 <= N <= 64:
        raise RuntimeError("A: 1 to 64 states per channel, not %d" % N)
    _check("B", B, ty, dev, (nb, T, N))
    _check("C", C, ty, dev, (nb, T, N))
    x, dt, B, C, A = _dense_last(x), _dense_last(dt), _dense_last(B), _dense_last(C), A.contiguous()
    zp = z_sb = z_st = 0
    if z is not None:
        _check("z", z, ty, dev, (nb, T, nd))
        z = _dense_last(z)
        zp, (z_sb, z_st, _) = z.data_ptr(), z.stride()
    Dp = bp = hp = 0
    if D is not None:
        _check("D", D, f32, dev, (nd,))
        D = D.contiguous()
        Dp = D.data_ptr()
    if dt_bias is not None:
        _check("dt_bias", dt_bias, f32, dev, (nd,))
        dt_bias = dt_bias.contiguous()
        bp = dt_bias.data_ptr()
    if state is not None:
        _check("state", state, f32, dev, (nb, N, nd))
        state = state.contiguous()
        hp = state.data_ptr()
    y = torch.empty((nb, T, nd), dtype=ty, device=dev)
    new = torch.empty((nb, N, nd), dtype=f32, device=dev)
    L = native.lib()
    need = L.rvm_selective_scan_workspace(nb, T, nd, N)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    xs, ds, Bs, Cs = x.stride(), dt.stride(), B.stride(), C.stride()
    _call(L.rvm_selective_scan, code,
          _SCAN.pack(x.data_ptr(), dt.data_ptr(), zp, B.data_ptr(), C.data_ptr(), A.data_ptr(), Dp, bp, hp, y.data_ptr(), new.data_ptr(),
                     ws.data_ptr() if ws is not None else 0, xs[0], xs[1], ds[0], ds[1], z_sb, z_st, Bs[0], Bs[1], Cs[0], Cs[1],
                     nb, T, nd, N, bool(softplus), need), dev)
    return y, new


def _paged(first, cache, table, lengths, offsets, code_of):
    """Checks of what append_kv and attend share; ``first`` is the tensor of the new rows."""
    code = _first(code_of, first)
    dev, dt = first.device, first.dtype
    if not (isinstance(cache, (tuple, list)) and len(cache) == 2):
        raise RuntimeError("cache must be the pair (key pages, value pages)")
    kp, vp = cache
    _check(code_of, first, dt, dev, (-1, -1, -1))
    _check("key pages", kp, dt, dev, (-1, -1, -1, first.shape[2]))
    _check("value pages", vp, dt, dev, kp.shape)
    if not (kp.is_contiguous() and vp.is_contiguous()):
        raise RuntimeError("the pages must be dense")
    _check("table", table, torch.int32, dev, (-1, -1))
    S = table.shape[0]
    _check("lengths", lengths, torch.int32, dev, (S,))
    if not (table.is_contiguous() and lengths.is_contiguous()):
        raise RuntimeError("table and lengths must be dense")
    op = 0
    if offsets is not None:
        _check("offsets", offsets, torch.int32, dev, (S + 1,))
        if not offsets.is_contiguous():
            raise RuntimeError("offsets must be dense")
        op = offsets.data_ptr()
    elif first.shape[0] != S:
        raise RuntimeError("without offsets every stream has one row: %d rows for %d streams" % (first.shape[0], S))
    return code, dev, dt, kp, vp, S, op


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
    code, dev, dt, kp, vp, S, op = _paged(k, cache, table, lengths, offsets, "k")
    M, Hkv, Dh = k.shape
    P, hk, page, _ = kp.shape
    _check("v", v, dt, dev, (M, Hkv, Dh))
    if hk != Hkv:
        raise RuntimeError("k has %d heads, the pages have %d" % (Hkv, hk))
    k, v = _rows(k), _rows(v)
    rot = fp = qp = op_q = q_sm = q_sh = 0
    Hq, out = Hkv, None
    if freqs is not None:
        _check("freqs", freqs, torch.float32, dev, (-1,))
        freqs = freqs.contiguous()
        rot, fp = 2 * freqs.numel(), freqs.data_ptr()
    if q is not None:
        _check("q", q, dt, dev, (M, -1, Dh))
        Hq = q.shape[1]
        q = _rows(q)
        out = torch.empty((M, Hq, Dh), dtype=dt, device=dev)
        qp, op_q, (q_sm, q_sh, _) = q.data_ptr(), out.data_ptr(), q.stride()
    if M and not S:
        raise RuntimeError("%d rows for no stream" % M)
    ks, vs = k.stride(), v.stride()
    _call(native.lib().rvm_append_kv, code,
          _APPEND.pack(qp, k.data_ptr(), v.data_ptr(), op_q, kp.data_ptr(), vp.data_ptr(), table.data_ptr(), lengths.data_ptr(), op, fp,
                       q_sm, q_sh, ks[0], ks[1], vs[0], vs[1], M, S, Hq, Hkv, Dh, P, page, table.shape[1], rot, bool(interleaved)), dev)
    return out


_ATTEND = struct.Struct("8P11qd")


def attend(q, cache, table, lengths, offsets=None, scale=None):
    """Attention of new tokens over their streams' caches: ``softmax_j(scale q . k_j) v_j`` over the positions up to the row's
    own, ``lengths[s] + i`` (the rows' own keys are appended first, with the same arguments).  ``q`` [M, heads, dim]; query
    head h reads key head ``h // (heads / kv heads)``; ``scale`` defaults to ``dim ** -0.5``.  Returns [M, heads, dim].

    A row with a negative position, or behind the last stream's rows, gives 0.  Pages outside the pool are not followed:
    a row that would read one gives NaN."""
    code, dev, dt, kp, vp, S, op = _paged(q, cache, table, lengths, offsets, "q")
    M, Hq, Dh = q.shape
    P, Hkv, page, _ = kp.shape
    if M and not S:
        raise RuntimeError("%d rows for no stream" % M)
    q = _rows(q)
    out = torch.empty((M, Hq, Dh), dtype=dt, device=dev)
    L = native.lib()
    scale = Dh ** -0.5 if scale is None else float(scale)
    sm, sh, _ = q.stride()
    head = (q.data_ptr(), kp.data_ptr(), vp.data_ptr(), out.data_ptr())
    tail = (table.data_ptr(), lengths.data_ptr(), op, sm, sh, M, S, Hq, Hkv, Dh, P, page, table.shape[1])
    need = L.rvm_attend_workspace(code, _ATTEND.pack(*head, 0, *tail, 0, scale))
    if need < 0:
        native.check(1, "rvm_attend_workspace")
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    _call(L.rvm_attend, code, _ATTEND.pack(*head, ws.data_ptr() if ws is not None else 0, *tail, need, scale), dev)
    return out
