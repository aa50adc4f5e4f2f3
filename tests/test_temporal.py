"""Temporal operators (causal convolution, selective scan, paged key-value cache and the attention over it) against 64-bit
restatements, with bounds derived from the number of roundings (oracle/temporal_oracle.py); refusals on the CPU."""
import ctypes
import os
import subprocess

import pytest
import torch

from oracle import temporal_oracle as O

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def _near(got, ref, bound, what):
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan), "%s: NaN in other places" % what
    off = torch.where(nan, torch.zeros_like(ref), (got - ref).abs() - bound)
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0, "%s: off by %.3g more than its bound" % (what, worst)


# ---- on the CPU ---------------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    from robustvideomatting_amd import temporal as M
    x = torch.zeros(1, 2, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        M.causal_conv(x, torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        M.selective_scan(x, x, torch.zeros(4, 8), x, x)
    pages = torch.zeros(1, 1, 16, 8)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        M.append_kv(torch.zeros(1, 1, 8), torch.zeros(1, 1, 8), (pages, pages), i[:, None], i)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        M.attend(torch.zeros(1, 1, 8), (pages, pages), i[:, None], i)


def test_tangents_are_refused():
    """Forward mode's dual tensors, which need no gradient: their tangents would be lost, under no_grad too."""
    import torch.autograd.forward_ad as F
    from robustvideomatting_amd import temporal as M
    x = torch.ones(2, 3)
    with F.dual_level():
        d = F.make_dual(x, x)
        M._tensor("x", x, x.dtype, x.device, (2, -1))
        assert not d.requires_grad and M._dual(None, x, d) and not M._dual(None, x)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match="x carries a tangent"):
                M._tensor("x", d, x.dtype, x.device, (2, -1))
        with torch.inference_mode():
            M._tensor("x", d, x.dtype, x.device, (2, -1))
    M._tensor("x", x, x.dtype, x.device, (2, -1))


def _refused(rc, text):
    from robustvideomatting_amd import native
    assert rc != 0 and text in native.lib().rvm_last_error().decode(), (rc, native.lib().rvm_last_error())


CONV_OK = dict(x=4096, weight=4096, bias=0, state_in=0, y=8192, state_out=12288, x_sb=8, x_st=8, B=1, T=1, D=8, W=4, silu=1)
SCAN_OK = dict(x=4096, dt=4096, z=0, B=4096, C=4096, A=4096, D=0, dt_bias=0, state_in=0, y=4096, state_out=4096, workspace=0, x_sb=8,
               x_st=8, dt_sb=8, dt_st=8, z_sb=0, z_st=0, B_sb=4, B_st=4, C_sb=4, C_st=4, nB=1, nT=1, nD=8, nN=4, softplus=1,
               workspace_bytes=0)
APPEND_OK = dict(q=4096, k=4096, v=4096, q_out=4096, k_pages=4096, v_pages=4096, table=4096, lengths=4096, offsets=0, freqs=4096, q_sm=64,
                 q_sh=16, k_sm=64, k_sh=16, v_sm=64, v_sh=16, M=2, S=2, Hq=4, Hkv=4, Dh=16, pages=2, page=16, width=1, rot=16,
                 interleaved=0)
ATTEND_OK = dict(q=4096, k_pages=4096, v_pages=4096, out=4096, workspace=0, table=4096, lengths=4096, offsets=0, q_sm=64, q_sh=16, M=2,
                 S=2, Hq=4, Hkv=4, Dh=16, pages=2, page=16, width=1, workspace_bytes=0, scale=0.25)


@pytest.mark.parametrize("entry,base,change,text", [
    ("rvm_causal_conv", CONV_OK, dict(W=5), "2 to 4 taps"),
    ("rvm_causal_conv", CONV_OK, dict(W=1), "2 to 4 taps"),
    ("rvm_causal_conv", CONV_OK, dict(B=-1), "shape"),
    ("rvm_causal_conv", CONV_OK, dict(T=1 << 31), "shape"),
    ("rvm_causal_conv", CONV_OK, dict(x=0), "null"),
    ("rvm_causal_conv", CONV_OK, dict(state_in=12288), "alias"),
    ("rvm_selective_scan", SCAN_OK, dict(nN=0), "states"),
    ("rvm_selective_scan", SCAN_OK, dict(nN=65), "states"),
    ("rvm_selective_scan", SCAN_OK, dict(A=0), "null"),
    ("rvm_selective_scan", SCAN_OK, dict(state_in=4096), "alias"),
    ("rvm_selective_scan", SCAN_OK, dict(nT=4096), "workspace"),
    ("rvm_selective_scan", SCAN_OK, dict(nD=-8), "shape"),
    ("rvm_append_kv", APPEND_OK, dict(Hq=3), "multiple"),
    ("rvm_append_kv", APPEND_OK, dict(Dh=20), "head size"),
    ("rvm_append_kv", APPEND_OK, dict(Dh=512), "head size"),
    ("rvm_append_kv", APPEND_OK, dict(page=24), "page size"),
    ("rvm_append_kv", APPEND_OK, dict(page=8), "page size"),
    ("rvm_append_kv", APPEND_OK, dict(M=3), "one row"),
    ("rvm_append_kv", APPEND_OK, dict(rot=8), "rotated"),
    ("rvm_append_kv", APPEND_OK, dict(rot=32), "rotated"),
    ("rvm_append_kv", APPEND_OK, dict(freqs=0), "null"),
    ("rvm_append_kv", APPEND_OK, dict(q=0), "null"),
    ("rvm_append_kv", APPEND_OK, dict(k=4098), "16-byte"),
    ("rvm_append_kv", APPEND_OK, dict(v_sh=13), "16-byte"),
    ("rvm_append_kv", APPEND_OK, dict(width=1 << 28), "pool or table"),
    ("rvm_append_kv", APPEND_OK, dict(pages=0), "pool or table"),
    ("rvm_attend", ATTEND_OK, dict(scale=0.0), "scale"),
    ("rvm_attend", ATTEND_OK, dict(scale=float("nan")), "scale"),
    ("rvm_attend", ATTEND_OK, dict(scale=-1.0), "scale"),
    ("rvm_attend", ATTEND_OK, dict(Hq=6), "multiple"),
    ("rvm_attend", ATTEND_OK, dict(lengths=0), "null"),
    ("rvm_attend", ATTEND_OK, dict(out=0), "null"),
    ("rvm_attend", ATTEND_OK, dict(q_sm=65), "16-byte"),
    ("rvm_attend", ATTEND_OK, dict(out=4104), "16-byte"),
])
def test_c_entries_refuse_bad_arguments_before_any_launch(entry, base, change, text):
    import struct
    from robustvideomatting_amd import native
    v = dict(base, **change)
    assert set(v) == set(base)
    block = struct.pack("%dqd" % (len(v) - 1) if "scale" in v else "%dq" % len(v), *v.values())
    _refused(getattr(native.lib(), entry)(0, block, None), text)


@pytest.mark.parametrize("entry,base,change,text", [
    ("rvm_causal_conv", CONV_OK, dict(B=1 << 20, T=1 << 20), "too large"),
    ("rvm_selective_scan", SCAN_OK, dict(nB=1 << 26), "too large"),
    ("rvm_selective_scan", SCAN_OK, dict(nB=1 << 20, nD=1 << 20), "too large"),
    ("rvm_append_kv", APPEND_OK, dict(M=1 << 24, S=1 << 24), "too large"),
    ("rvm_append_kv", APPEND_OK, dict(Hkv=4096, Hq=4096, page=1024, Dh=256, pages=1), "below 2 GiB"),
    ("rvm_attend", ATTEND_OK, dict(M=1 << 24, S=1 << 24), "too large"),
    ("rvm_attend", ATTEND_OK, dict(M=1 << 20, S=8, offsets=4096, Hq=4096), "too large"),
    ("rvm_attend", ATTEND_OK, dict(M=8, S=1 << 21, offsets=4096, Hq=8, Hkv=8), "too large"),
    ("rvm_attend", ATTEND_OK, dict(M=1 << 21, S=1 << 20, offsets=4096, Hq=260, Hkv=4), "too large"),
    ("rvm_attend", ATTEND_OK, dict(M=1 << 20, S=1 << 20, Hq=1024), "too large"),
    ("rvm_attend", ATTEND_OK, dict(Hkv=8192, Hq=8192, page=1024, Dh=128), "below 2 GiB"),
    ("rvm_attend", ATTEND_OK, dict(width=64), "workspace"),
    ("rvm_attend", ATTEND_OK, dict(width=64, offsets=4096), "workspace"),
    ("rvm_attend", ATTEND_OK, dict(width=64, workspace=4104, workspace_bytes=1 << 40), "workspace"),
])
def test_c_entries_refuse_what_no_launch_holds(entry, base, change, text):
    import struct
    from robustvideomatting_amd import native
    v = dict(base, **change)
    assert set(v) == set(base)
    block = struct.pack("%dqd" % (len(v) - 1) if "scale" in v else "%dq" % len(v), *v.values())
    _refused(getattr(native.lib(), entry)(0, block, None), text)


def test_scan_rows_past_32_bit_offsets_are_refused():
    """fp32 rows of more than 4 GiB."""
    import struct
    from robustvideomatting_amd import native
    v = dict(SCAN_OK, nD=(1 << 30) + 1, nN=1)
    _refused(native.lib().rvm_selective_scan(0, struct.pack("%dq" % len(v), *v.values()), None), "too large")


@pytest.mark.parametrize("scale", [3e38, 1e39, 1e300, float("inf"), 1e-46, 1e-300, -1e-50])
def test_scales_outside_fp32_are_refused(scale):
    """The kernels scale in fp32 (and in base 2): infinite there, or 0, which a masked score would turn into NaN."""
    import struct
    from robustvideomatting_amd import native
    v = dict(ATTEND_OK, scale=scale)
    _refused(native.lib().rvm_attend(0, struct.pack("%dqd" % (len(v) - 1), *v.values()), None), "scale")


@pytest.mark.parametrize("entry,base", [("rvm_append_kv", APPEND_OK), ("rvm_attend", ATTEND_OK)])
def test_c_entries_refuse_rows_for_no_stream(entry, base):
    """No stream, but rows: refused rather than left as they were.  Neither rows nor streams: nothing to do."""
    import struct
    from robustvideomatting_amd import native
    pack = lambda v: struct.pack("%dqd" % (len(v) - 1) if "scale" in v else "%dq" % len(v), *v.values())
    rows = pack(dict(base, S=0, offsets=4096))
    _refused(getattr(native.lib(), entry)(0, rows, None), "no stream")
    if entry == "rvm_attend":
        assert native.lib().rvm_attend_workspace(0, rows) == -1
    assert getattr(native.lib(), entry)(0, pack(dict(base, S=0, M=0)), None) == 0
    assert getattr(native.lib(), entry)(0, pack(dict(base, S=2, M=0, offsets=4096)), None) == 0


def test_positions_and_keys_stay_inside_an_int(tmp_path):
    """A stream's positions saturate instead of wrapping round, and a pass over its keys ends one behind the table."""
    src = tmp_path / "pos.cpp"
    src.write_text('#include "%s/robustvideomatting_amd/csrc/paged_index.hpp"\nextern "C" int at(int l, int i) { return paged_position(l, i); }\n'
                   'extern "C" unsigned keys(int w, int sh, int pos) { return paged_keys(w, sh, pos); }\n' % ROOT)
    lib = tmp_path / "pos.so"
    subprocess.check_call(["g++", "-O1", "-shared", "-fPIC", "-o", str(lib), str(src)])
    f = ctypes.CDLL(str(lib))
    f.keys.restype = ctypes.c_uint
    top = 2 ** 31 - 1
    assert [f.at(0, 0), f.at(7, 5), f.at(-3, 2), f.at(-3, 3), f.at(top, 0), f.at(top, 9), f.at(-top - 1, 0)] == [0, 12, -1, 0, top, top, -top - 1]
    assert [f.keys(3, 4, p) for p in (0, 46, 47, 48, 100, top)] == [1, 47, 48, 49, 49, 49]
    assert [f.keys(1 << 21, 10, p) for p in (0, top - 1, top)] == [1, top, top + 1]


def test_c_entries_refuse_bad_types_and_null():
    from robustvideomatting_amd import native
    L = native.lib()
    for name in ("rvm_causal_conv", "rvm_selective_scan", "rvm_append_kv", "rvm_attend"):
        _refused(getattr(L, name)(7, b"\0" * 512, None), "dtype")
        _refused(getattr(L, name)(0, None, None), "null")
    assert L.rvm_attend_workspace(9, b"\0" * 512) == -1
    assert L.rvm_selective_scan_workspace(1, 1, 1, 65) == -1 and L.rvm_selective_scan_workspace(-1, 1, 1, 1) == -1


def test_page_lookup_stays_inside_the_table_and_the_pool(tmp_path):
    """The lookup every kernel goes through, on the host: columns past the table and pages outside the pool are -1."""
    src = tmp_path / "page_of.cpp"
    src.write_text('#include "%s/robustvideomatting_amd/csrc/paged_index.hpp"\nextern "C" int look(const int* t, int w, int p, int sh, int s, int pos)'
                   ' { return page_of(t, w, p, sh, s, pos); }\n' % ROOT)
    lib = tmp_path / "page_of.so"
    subprocess.check_call(["g++", "-O1", "-shared", "-fPIC", "-o", str(lib), str(src)])
    look = ctypes.CDLL(str(lib)).look
    t = (ctypes.c_int * 6)(3, -1, 7, 8, 2 ** 31 - 1, 0)         # two streams of three columns, a pool of eight pages
    at = lambda s, pos: look(t, 3, 8, 4, s, pos)
    assert [at(0, p) for p in (0, 15, 16, 31, 32, 47)] == [3, 3, -1, -1, 7, 7]
    assert [at(1, p) for p in (0, 16, 32)] == [-1, -1, 0]
    assert [at(1, p) for p in (48, 2 ** 31 - 1, -1, -16)] == [-1] * 4


def _scan_index(tmp_path):
    src = tmp_path / "scan_index.cpp"
    src.write_text('#include "%s/robustvideomatting_amd/csrc/scan_index.hpp"\nextern "C" {\nint batch(int np, int pack) { return scan_batch(np, pack); }\n'
                   'int values(int np, int ends) { return scan_values(np, ends); }\nint loads(int np, int pack, int ends) { return scan_loads(np, pack, ends); }\n'
                   'int step_of(int e, int np, int pack, int ends) { return scan_step_of(e, np, pack, ends); }\n'
                   'long long chunk_len(long long t, long long n) { return scan_chunk_len(t, n); }\nint first(int t, int len, int ch) { return scan_first_step(t, len, ch); }\n'
                   'int end(int t, int len, int first) { return scan_end_step(t, len, first); }\n}\n' % ROOT)
    lib = tmp_path / "scan_index.so"
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(lib), str(src)])
    return ctypes.CDLL(str(lib))


@pytest.mark.parametrize("states", [8, 16, 32, 64])
@pytest.mark.parametrize("pack", [1, 2, 4])
@pytest.mark.parametrize("ends", [0, 1])
def test_scan_lanes_stay_inside_their_batch(tmp_path, states, pack, ends):
    """What a wave requests of B and C: every value of the batch, each at its place, and no step behind the batch - also
    where the batch has fewer values than the wave has lanes."""
    f = _scan_index(tmp_path)
    batch, values, loads = f.batch(states, pack), f.values(states, ends), f.loads(states, pack, ends)
    assert (loads - 1) * 64 < batch * pack * values <= loads * 64
    steps = [f.step_of(e, states, pack, ends) for e in range(loads * 64)]
    assert steps[:batch * pack * values] == [k for k in range(batch) for _ in range(pack * values)]
    assert 0 <= min(steps) and max(steps) == batch - 1


@pytest.mark.parametrize("T,D,N", [(40, 8, 16), (63, 8, 4), (1021, 333, 13), (8160, 960, 16), (2 ** 31 - 65, 1, 1), (2 ** 31 - 65, 64, 1),
                                   (2 ** 31 - 16385, 33, 64), (2 ** 31 - 16383, 64, 8), (2 ** 31 - 65, 900, 1)])
def test_scan_chunks_cover_every_step_once(tmp_path, T, D, N):
    """The chunks that a length is cut into, up to the longest that the entry takes: end to end, from 0 to T."""
    from robustvideomatting_amd import native
    f = _scan_index(tmp_path)
    f.chunk_len.restype = ctypes.c_longlong
    f.chunk_len.argtypes = [ctypes.c_longlong] * 2
    need = native.lib().rvm_selective_scan_workspace(1, T, D, N)
    chunks = need // 4 // ((N + 1) * D) * 8 // 9                # a slot a chunk, and one for every eight
    assert chunks >= 8 and chunks % 8 == 0 and chunks * 9 // 8 * (N + 1) * D * 4 == need
    length, at = f.chunk_len(T, chunks), 0
    assert 0 < length < 2 ** 31
    for ch in range(chunks):
        first, end = f.first(T, length, ch), f.end(T, length, f.first(T, length, ch))
        assert first == at and first <= end <= T, ch
        at = end
    assert at == T


# ---- convolution --------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,T,D,W,bias,state,silu,sliced", [
    (1, 1, 8, 4, True, True, True, False), (3, 1, 5, 4, True, True, True, False), (2, 2, 24, 4, False, True, True, False),
    (2, 3, 64, 3, True, False, False, True), (1, 16, 960, 4, True, True, True, True), (2, 17, 33, 2, True, True, True, True),
    (5, 100, 40, 4, True, True, True, False), (2, 0, 16, 4, True, True, True, False), (1, 257, 1, 4, False, False, True, False),
])
def test_causal_conv(dtype, B, T, D, W, bias, state, silu, sliced):
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(B * 100 + T + D)
    x = _rn(g, B, T, 2 * D + 3, dtype=dt)[..., 3:D + 3] if sliced else _rn(g, B, T, D, dtype=dt)
    w = _rn(g, W, D, dtype=dt)
    b = _rn(g, D, dtype=dt) if bias else None
    s = _rn(g, B, W - 1, D, dtype=dt) if state else None
    y, new = M.causal_conv(x, w, b, state=s, silu=silu)
    (ry, rs), bound = O.causal_conv(x, w, b, s, silu)
    assert y.dtype == new.dtype == dt
    assert torch.equal(new.double(), rs)
    _near(y, ry, O.rounded(ry, bound, dt), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D,front", [(20, 0), (20, 4), (26, 0), (26, 2), (40, 1), (40, 4), (64, 2)])
def test_causal_conv_pieces(dtype, D, front):
    """Channels and rows that begin on every kind of boundary: pieces of 16 bytes and fewer, single steps and runs."""
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(D + front)
    for T in (1, 21):
        x = _rn(g, 3, T, 2 * D, dtype=dt)[..., front:D + front]
        w, b, s = _rn(g, 4, D, dtype=dt), _rn(g, D, dtype=dt), _rn(g, 3, 3, D, dtype=dt)
        y, new = M.causal_conv(x, w, b, state=s)
        (ry, rs), bound = O.causal_conv(x, w, b, s, True)
        assert torch.equal(new.double(), rs)
        _near(y, ry, O.rounded(ry, bound, dt), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_a_chunk_equals_its_steps(dtype):
    """One call with T steps gives the bits of T calls with one step: convolution and scan."""
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(5)
    B, T, D, N, W = 2, 7, 40, 16, 4
    x, w, b = _rn(g, B, T, D, dtype=dt), _rn(g, W, D, dtype=dt), _rn(g, D, dtype=dt)
    step, Bm, Cm, z = _rn(g, B, T, D, dtype=dt), _rn(g, B, T, N, dtype=dt), _rn(g, B, T, N, dtype=dt), _rn(g, B, T, D, dtype=dt)
    A, Dv, db = -_rn(g, N, D).abs(), _rn(g, D), _rn(g, D)
    y, cs = M.causal_conv(x, w, b)
    o, hs = M.selective_scan(y, step, A, Bm, Cm, Dv, z, db)
    c1 = h1 = None
    for t in range(T):
        y1, c1 = M.causal_conv(x[:, t:t + 1], w, b, state=c1)
        o1, h1 = M.selective_scan(y1, step[:, t:t + 1], A, Bm[:, t:t + 1], Cm[:, t:t + 1], Dv, z[:, t:t + 1], db, state=h1)
        assert torch.equal(y1[:, 0], y[:, t]) and torch.equal(o1[:, 0], o[:, t]), t
    assert torch.equal(c1, cs) and torch.equal(h1, hs)


# ---- scan ---------------------------------------------------------------------------------------------------------------
def _scan_inputs(g, B, T, D, N, dt, sliced=False):
    x = _rn(g, B, T, D, dtype=dt)
    step = _rn(g, B, T, D + 1, dtype=dt, scale=0.5)[..., 1:] if sliced else _rn(g, B, T, D, dtype=dt, scale=0.5)
    bc = _rn(g, B, T, 2 * N + 1, dtype=dt)
    A = -(torch.arange(1, N + 1).float()[:, None] * torch.exp(0.3 * torch.randn((N, D), generator=g))).cuda()
    bias = (torch.rand(D, generator=g) * 6 - 7).cuda()              # step sizes from 1e-3 to 0.3
    return x, step, A, bc[..., :N], bc[..., N:2 * N], _rn(g, D), bias


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,T,D,N,z,state,sliced", [
    (1, 1, 1, 1, False, False, False), (2, 1, 64, 16, True, True, False), (3, 2, 65, 16, True, True, True), (1, 9, 33, 13, False, True, True),
    (2, 40, 100, 8, True, False, False), (1, 33, 24, 64, True, True, False), (4, 65, 7, 24, True, True, True), (1, 300, 960, 16, True, True, False),
    (1, 2049, 70, 16, True, True, True), (2, 1500, 130, 4, False, False, False), (40, 130, 64, 16, True, True, False), (2, 0, 16, 16, True, True, False),
    (1, 4100, 16, 32, True, True, False),
])
def test_selective_scan(dtype, B, T, D, N, z, state, sliced):
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(B + T + D + N)
    x, step, A, Bm, Cm, Dv, bias = _scan_inputs(g, B, T, D, N, dt, sliced)
    zz = _rn(g, B, T, 2 * D, dtype=dt)[..., D:] if z else None
    h0 = _rn(g, B, N, D) if state else None
    keep = h0.clone() if state else None
    y, h = M.selective_scan(x, step, A, Bm, Cm, Dv, zz, bias, h0)
    (ry, rh), (by, bh) = O.selective_scan(x, step, A, Bm, Cm, Dv, zz, bias, h0)
    assert y.dtype == dt and h.dtype == torch.float32
    _near(h, rh, bh + 1e-37, "state")
    _near(y, ry, O.rounded(ry, by, dt), "y")
    assert not state or torch.equal(h0, keep)
    again = M.selective_scan(x, step, A, Bm, Cm, Dv, zz, bias, h0)
    assert torch.equal(again[0], y) and torch.equal(again[1], h)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,T,D,N,state,sliced", [
    (4099, 1, 16, 16, True, False), (4098, 2, 20, 24, True, True), (1031, 40, 7, 8, True, True), (131, 300, 13, 16, True, True),
    (67, 500, 31, 32, False, True), (133, 257, 32, 5, True, False), (1, 8160, 16, 16, True, False), (4097, 3, 1, 1, False, False),
    (600, 64, 32, 64, True, False),
])
def test_selective_scan_of_many_narrow_sequences(dtype, B, T, D, N, state, sliced):
    """Fewer channels than lanes and many sequences, whose number no group of them divides."""
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(B + T + D + N)
    x, step, A, Bm, Cm, Dv, bias = _scan_inputs(g, B, T, D, N, dt, sliced)
    zz = _rn(g, B, T, 2 * D, dtype=dt)[..., D:] if sliced else None
    h0 = _rn(g, B, N, D) if state else None
    y, h = M.selective_scan(x, step, A, Bm, Cm, Dv, zz, bias, h0)
    (ry, rh), (by, bh) = O.selective_scan(x, step, A, Bm, Cm, Dv, zz, bias, h0)
    _near(h, rh, bh + 1e-37, "state")
    _near(y, ry, O.rounded(ry, by, dt), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [39, 40, 41, 47, 63, 64, 65, 95, 96, 97])
def test_selective_scan_around_the_first_chunks(T):
    """Lengths at which the time axis begins to be cut, and chunks that are empty or shorter than the others."""
    from robustvideomatting_amd import temporal as M
    for B, D, N in ((2, 70, 16), (1, 33, 64), (550, 64, 8)):
        g = _gen(T + B)
        x, step, A, Bm, Cm, Dv, bias = _scan_inputs(g, B, T, D, N, torch.bfloat16, True)
        h0 = _rn(g, B, N, D)
        y, h = M.selective_scan(x, step, A, Bm, Cm, Dv, None, bias, h0)
        (ry, rh), (by, bh) = O.selective_scan(x, step, A, Bm, Cm, Dv, None, bias, h0)
        _near(h, rh, bh + 1e-37, "state")
        _near(y, ry, O.rounded(ry, by, torch.bfloat16), "y")


@pytest.mark.gpu
def test_selective_scan_without_softplus_and_options():
    from robustvideomatting_amd import temporal as M
    g = _gen(3)
    x, step, A, Bm, Cm, Dv, bias = _scan_inputs(g, 2, 50, 30, 16, torch.float32)
    step = step.abs() * 0.1
    y, h = M.selective_scan(x, step, A, Bm, Cm, softplus=False)
    (ry, rh), (by, bh) = O.selective_scan(x, step, A, Bm, Cm, softplus=False)
    _near(h, rh, bh, "state")
    _near(y, ry, O.rounded(ry, by, torch.float32), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 3000])
def test_scan_large_and_tiny_step_sizes(T):
    """Steps that forget everything at once, and steps so small that exp(v) is below half a unit of 1."""
    from robustvideomatting_amd import temporal as M
    g = _gen(9)
    x, step, A, Bm, Cm, Dv, _ = _scan_inputs(g, 1, T, 48, 16, torch.float32)
    bias = torch.linspace(-25, 40, 48).cuda()
    h0 = _rn(g, 1, 16, 48)
    y, h = M.selective_scan(x, step, A, Bm, Cm, Dv, None, bias, h0)
    (ry, rh), (by, bh) = O.selective_scan(x, step, A, Bm, Cm, Dv, None, bias, h0)
    _near(h, rh, bh + 1e-37, "state")
    _near(y, ry, O.rounded(ry, by, torch.float32), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("sign,softplus", [(1.0, False), (-1.0, False), (1.0, True)])
@pytest.mark.parametrize("B,D,N", [(1, 70, 4), (2, 33, 16), (1, 40, 40)])
def test_scan_states_that_grow_past_a_factor_s_range(dtype, sign, softplus, B, D, N):
    """A stream's steps multiply a state by e^145, more than fp32 holds: one that is zero stays zero until its first input,
    and a tiny one becomes a large one, where the time axis is cut and where it is not."""
    from robustvideomatting_amd import temporal as M
    dt, g, T = DT[dtype], _gen(N), 100
    x, Bm, Cm = torch.zeros((B, T, D), dtype=dt, device="cuda"), _rn(g, B, T, N, dtype=dt), _rn(g, B, T, N, dtype=dt)
    x[:, 90:, :D // 2] = _rn(g, B, 10, D // 2, dtype=dt)
    h0 = _rn(g, B, N, D) * 1e-35
    h0[..., :D // 2] = 0
    A = torch.full((N, D), 1.45 * sign, device="cuda")
    A[1::2] *= -0.5                                         # beside states that decay
    step = torch.full((B, T, D), sign * (0.5 if softplus else 1.0), dtype=dt, device="cuda")
    bias = torch.full((D,), 0.04, device="cuda") if softplus else None
    y, h = M.selective_scan(x, step, A, Bm, Cm, None, None, bias, h0, softplus=softplus)
    (ry, rh), (by, bh) = O.selective_scan(x, step, A, Bm, Cm, None, None, bias, h0, softplus=softplus)
    assert torch.isfinite(rh).all() and rh.abs().max() > 1e24 and not ry[:, :90, :D // 2].any()
    _near(h, rh, bh + 1e-37, "state")
    _near(y, ry, O.rounded(ry, by, dt), "y")
    for t in range(T):                                      # step by step
        y1, h0 = M.selective_scan(x[:, t:t + 1], step[:, t:t + 1], A, Bm[:, t:t + 1], Cm[:, t:t + 1], None, None, bias, h0, softplus=softplus)
    _near(h0, rh, bh + 1e-37, "state, step by step")


# ---- paged cache --------------------------------------------------------------------------------------------------------
def _paged(g, lengths, new, Hkv, Dh, page, dt, spare=2, fill=0.0):
    """Pools whose pages are dealt out at random; a table with room; -> (cache, table tensor, table list, lengths tensor)"""
    need = [max(0, -(-(p + n) // page)) for p, n in zip(lengths, new)]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g).tolist()
    width = max(need + [1]) + 1
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [pool + 5] * (width - n))        # what is not dealt out is outside the pool
        at += n
    cache = (torch.full((pool, Hkv, page, Dh), fill, dtype=dt, device="cuda"), torch.full((pool, Hkv, page, Dh), fill, dtype=dt, device="cuda"))
    return cache, torch.tensor(rows, dtype=torch.int32).cuda(), rows, torch.tensor(lengths, dtype=torch.int32).cuda()


def _offsets(new):
    o = [0]
    for n in new:
        o.append(o[-1] + n)
    return o


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("lengths,new,Hq,Hkv,Dh,page,rot,inter,tail", [
    ([0], [1], 1, 1, 8, 16, 0, False, 0), ([5, 0, 300], [1, 1, 1], 4, 2, 64, 16, 64, False, 0), ([15, 16, 17], [3, 0, 40], 8, 2, 128, 16, 128, False, 0),
    ([0, 100], [33, 70], 3, 3, 80, 32, 48, True, 0), ([-2, 7, -9], [5, 1, 4], 2, 1, 32, 16, 16, False, 3), ([1000003], [2], 2, 2, 96, 1024, 96, True, 0),
    ([0] * 130, [1] * 130, 2, 1, 16, 16, 16, False, 0), ([3] * 70, [2] * 70, 1, 1, 24, 64, 16, True, 1), ([4, 9], [600, 3], 5, 1, 256, 128, 256, False, 0),
])
def test_append_kv(dtype, lengths, new, Hq, Hkv, Dh, page, rot, inter, tail):
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(sum(new) + Dh)
    cache, table, rows, lens = _paged(g, lengths, new, Hkv, Dh, page, dt, fill=7.0)
    off = _offsets(new)
    R = off[-1] + tail
    qkv = _rn(g, R, Hq + 2 * Hkv, Dh, dtype=dt)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    freqs = (10000.0 ** (-torch.arange(0, rot, 2).float() / max(rot, 1))).cuda() if rot else None
    one = all(n == 1 for n in new) and not tail
    offsets = None if one else torch.tensor(off, dtype=torch.int32).cuda()
    out = M.append_kv(k, v, cache, table, lens, offsets, freqs=freqs, q=q, interleaved=inter)
    want_k, want_v = (torch.full(cache[0].shape, 7.0, dtype=torch.float64, device="cuda") for _ in range(2))
    bk, wq, bq = torch.zeros_like(want_k), torch.zeros((R, Hq, Dh), dtype=torch.float64, device="cuda"), torch.zeros((R, Hq, Dh), dtype=torch.float64, device="cuda")
    turn = (lambda x, p: O.rotate(x, p, freqs, inter)) if rot else (lambda x, p: (x.double(), torch.zeros_like(x.double())))
    for m, (s, pos) in enumerate(O.rows_of(R, lengths, None if one else off)):
        if s is None:
            continue
        wq[m], bq[m] = turn(q[m], pos)
        if pos < 0:
            continue
        pg = rows[s][pos // page]
        want_k[pg, :, pos % page], bk[pg, :, pos % page] = turn(k[m], pos)
        want_v[pg, :, pos % page] = v[m].double()
    assert torch.equal(cache[1].double(), want_v)
    plain = rot if rot else 0
    assert torch.equal(cache[0].double()[..., plain:], want_k[..., plain:])
    _near(cache[0], want_k, O.rounded(want_k, bk, dt), "keys")
    _near(out, wq, O.rounded(wq, bq, dt), "q")


@pytest.mark.gpu
def test_append_without_q_and_far_positions():
    """Positions near 2^31: the angle keeps its digits.  The table of such a stream is long; its last page is looked up."""
    from robustvideomatting_amd import temporal as M
    g, page, pos = _gen(1), 1024, 2 ** 31 - 2000
    width = 2 ** 21
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, pos // page] = 1
    cache = (torch.zeros((2, 1, page, 16), device="cuda"), torch.zeros((2, 1, page, 16), device="cuda"))
    k, v = _rn(g, 1, 1, 16), _rn(g, 1, 1, 16)
    freqs = (10000.0 ** (-torch.arange(0, 16, 2).float() / 16)).cuda()
    assert M.append_kv(k, v, cache, table, torch.tensor([pos], dtype=torch.int32).cuda(), freqs=freqs) is None
    want, bound = O.rotate(k[0], pos, freqs)
    # 64-bit angle: 2^31 x 1 rad is held to 2^-22, and both sides round it
    _near(cache[0][1, :, pos % page], want, O.rounded(want, bound + 2.0 ** -20 * k[0].abs().sum().double(), torch.float32), "keys")
    assert torch.equal(cache[1][1, :, pos % page], v[0])


@pytest.mark.gpu
def test_append_drops_tokens_without_a_page():
    from robustvideomatting_amd import temporal as M
    cache = (torch.zeros((2, 1, 16, 16), device="cuda"), torch.zeros((2, 1, 16, 16), device="cuda"))
    table = torch.tensor([[2], [-1], [2 ** 31 - 1], [1], [0]], dtype=torch.int32).cuda()
    lens = torch.tensor([0, 3, 5, 16, 4], dtype=torch.int32).cuda()         # the fourth is past its table, the last is fine
    k = torch.ones((5, 1, 16), device="cuda")
    M.append_kv(k, k, cache, table, lens)
    assert cache[0].sum() == 16 and cache[1].sum() == 16 and (cache[0][0, 0, 4] == 1).all()


# ---- attention ----------------------------------------------------------------------------------------------------------
def _attend_case(g, lengths, new, Hq, Hkv, Dh, page, dt, fill, scale=1.0):
    cache, table, rows, lens = _paged(g, lengths, new, Hkv, Dh, page, dt, fill=fill)
    for s, (p, n) in enumerate(zip(lengths, new)):
        for pos0 in range(0, max(0, p + n), page):
            c = min(page, p + n - pos0)
            pg = rows[s][pos0 // page]
            cache[0][pg, :, :c] = _rn(g, Hkv, c, Dh, dtype=dt, scale=scale)
            cache[1][pg, :, :c] = _rn(g, Hkv, c, Dh, dtype=dt)
    return cache, table, rows, lens


ATTEND = [
    # lengths, new, Hq, Hkv, Dh, page
    ([0], [1], 1, 1, 8, 16), ([0, 1, 15, 16, 17], [1] * 5, 4, 4, 64, 16), ([300, 31, -1, 63], [1] * 4, 8, 2, 64, 16),
    ([2000, 5], [1, 1], 32, 4, 128, 64), ([700], [1], 5, 1, 80, 32), ([129, 64], [1, 1], 24, 3, 256, 128), ([4000], [1], 16, 1, 96, 1024),
    ([0], [33], 2, 1, 64, 16), ([0, 7, 40], [70, 0, 129], 8, 2, 128, 64), ([10, 200], [3, 2], 4, 4, 32, 16), ([-5, 90], [20, 40], 6, 2, 80, 32),
    ([1000], [65], 3, 3, 96, 128), ([0, 0, 0, 513], [1, 300, 2, 31], 4, 1, 64, 16), ([3000], [4], 8, 8, 128, 64), ([17], [260], 1, 1, 200, 16),
    ([100, 2000, 33], [1, 1, 1], 24, 1, 64, 16), ([5000, 0, 700], [1] * 3, 40, 2, 128, 64), ([900, 1200], [1, 1], 4, 4, 256, 256),
    ([40], [50], 24, 1, 64, 32), ([0] * 70, [3] * 70, 2, 2, 32, 16), ([250, -40, 3], [16, 16, 16], 16, 16, 40, 32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("lengths,new,Hq,Hkv,Dh,page", ATTEND)
def test_attend(dtype, lengths, new, Hq, Hkv, Dh, page):
    """Slots that hold no token hold NaN: nothing of them may reach a result."""
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(sum(new) + sum(lengths) + Dh)
    cache, table, rows, lens = _attend_case(g, lengths, new, Hq, Hkv, Dh, page, dt, float("nan"))
    off = _offsets(new)
    one = all(n == 1 for n in new)
    tail = 0 if one else 2
    q = _rn(g, off[-1] + tail, Hq + 1, Dh, dtype=dt)[:, 1:]
    offsets = None if one else torch.tensor(off, dtype=torch.int32).cuda()
    got = M.attend(q, cache, table, lens, offsets)
    ref, bound = O.attend(q, *cache, rows, lengths, None if one else off)
    _near(got, ref, O.rounded(ref, bound, dt), "out")
    assert torch.equal(M.attend(q, cache, table, lens, offsets), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("lengths,new,Hq,Hkv,Dh,page", [
    ([6000], [4], 2, 2, 64, 64), ([3000, 0, 50, 2000, -20, 700], [5, 300, 0, 64, 40, 1], 6, 2, 80, 16), ([2500, 1600], [130, 33], 40, 40, 32, 32),
    ([47 * i % 1700 - 40 for i in range(32)], [2] * 32, 4, 1, 64, 64), ([47 * i % 1700 - 40 for i in range(33)], [2] * 33, 4, 1, 64, 64),
    ([1900, 4, 1900], [20, 700, 20], 8, 1, 200, 128), ([3000, 10, 900], [140, 140, 140], 300, 2, 16, 64),
])
def test_attend_chunks_in_parts(dtype, lengths, new, Hq, Hkv, Dh, page):
    """Long keys behind few rows beside short ones: row tiles that are cut into parts, and others that are not."""
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(sum(new) + Dh)
    cache, table, rows, lens = _attend_case(g, lengths, new, Hq, Hkv, Dh, page, dt, float("nan"))
    off = _offsets(new)
    q = _rn(g, off[-1], Hq, Dh, dtype=dt)
    got = M.attend(q, cache, table, lens, torch.tensor(off, dtype=torch.int32).cuda())
    ref, bound = O.attend(q, *cache, rows, lengths, off)
    _near(got, ref, O.rounded(ref, bound, dt), "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("longest", [60, 3000])
def test_attend_one_token_rounds_once(dtype, longest):
    """One token a stream, 16-bit: the result is that of 32 bits, rounded once - the weights keep their digits."""
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(longest + 1)
    for Hq, Hkv, Dh in ((8, 2, 64), (6, 3, 128), (2, 2, 256)):
        lengths = [0, 1, 7, 31, 40, longest]
        cache, table, rows, lens = _attend_case(g, lengths, [1] * 6, Hq, Hkv, Dh, 16, dt, float("nan"))
        q = _rn(g, 6, Hq, Dh, dtype=dt)
        got = M.attend(q, cache, table, lens)
        ref, bound = O.attend(q, *cache, rows, lengths, parts=2)
        _near(got, ref, O.rounded(ref, bound, dt), "out, heads of %d" % Dh)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("longest", [100, 3000])
def test_attend_one_token_with_values_that_are_not_finite(dtype, bad, longest):
    """A value that is not finite decides its own dim, for the heads that read it, and touches no other - in a segment that a block
    has whole, and in one that is put together from pieces."""
    from robustvideomatting_amd import temporal as M
    dt, g, lengths = DT[dtype], _gen(17), [longest, 20]
    cache, table, rows, lens = _attend_case(g, lengths, [1, 1], 4, 2, 64, 16, dt, 0.0)
    q = _rn(g, 2, 4, 64, dtype=dt)
    clean, bound = O.attend(q, *cache, rows, lengths, parts=2 if dt != torch.float32 else 1)
    for at, dim in ((0, 0), (37, 5), (longest, 63)):
        cell = cache[1][rows[0][at // 16], 1, at % 16]
        keep = cell[dim].item()
        cell[dim] = bad
        got = M.attend(q, cache, table, lens)
        cell[dim] = keep
        want = clean.clone()
        want[0, 2:, dim] = bad
        hit = torch.zeros_like(want, dtype=torch.bool)
        hit[0, 2:, dim] = True
        assert torch.equal(got[hit].double().nan_to_num(7.0), want[hit].nan_to_num(7.0)), (at, got[hit])
        got[hit] = 0
        want[hit] = 0
        _near(got, want, O.rounded(want, bound, dt), "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("new", [[1, 1], [40, 3], [300, 17]])
def test_attend_large_scores_and_scale(dtype, new):
    """Scores in the hundreds (weights of nearly 0 and 1), another scale than the default."""
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(sum(new))
    lengths = [200, 1]
    cache, table, rows, lens = _attend_case(g, lengths, new, 4, 2, 64, 16, dt, 0.0, scale=16.0)
    off = _offsets(new)
    one = new == [1, 1]
    q = _rn(g, off[-1], 4, 64, dtype=dt, scale=4.0)
    got = M.attend(q, cache, table, lens, None if one else torch.tensor(off, dtype=torch.int32).cuda(), scale=0.3)
    ref, bound = O.attend(q, *cache, rows, lengths, None if one else off, scale=0.3)
    _near(got, ref, O.rounded(ref, bound, dt), "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, bad):
    """Keys and values of later tokens of the same chunk hold NaN or infinities: earlier rows are what they are without them."""
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(8)
    for lengths, new, at in (([0], [90], 50), ([70], [40], 80), ([500, 0], [64, 300], 520)):
        cache, table, rows, lens = _attend_case(g, lengths, new, 4, 2, 64, 16, dt, 0.0)
        off = _offsets(new)
        q = _rn(g, off[-1], 4, 64, dtype=dt)
        offsets = torch.tensor(off, dtype=torch.int32).cuda()
        clean = M.attend(q, cache, table, lens, offsets)
        pg, slot = rows[0][at // 16], at % 16
        for which in (0, 1):
            keep = cache[which][pg, :, slot].clone()
            cache[which][pg, :, slot] = bad
            got = M.attend(q, cache, table, lens, offsets)
            first = at - lengths[0]                         # the first row that sees the position
            assert torch.equal(got[:first], clean[:first]) and torch.equal(got[off[1]:], clean[off[1]:]), which
            ref, _ = O.attend(q[first:off[1]], *cache, rows[:1], [at], [0, off[1] - first])
            fin = torch.isfinite(ref)
            assert torch.equal(torch.isfinite(got[first:off[1]]), fin), which
            cache[which][pg, :, slot] = keep


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1, 1, 1], [50, 20, 3]])
def test_attend_does_not_follow_bad_pages(new):
    from robustvideomatting_amd import temporal as M
    g, lengths = _gen(4), [100, 70, 40]
    cache, table, rows, lens = _attend_case(g, lengths, new, 4, 2, 64, 16, torch.bfloat16, 0.0)
    for s, c, v in ((0, 5, -3), (1, 4, 2 ** 31 - 1)):
        rows[s][c] = v
        table[s, c] = v
    off = _offsets(new)
    one = new == [1, 1, 1]
    q = _rn(g, off[-1], 4, 64, dtype=torch.bfloat16)
    got = M.attend(q, cache, table, lens, None if one else torch.tensor(off, dtype=torch.int32).cuda())
    ref, bound = O.attend(q, *cache, rows, lengths, None if one else off)
    assert torch.isnan(ref[:off[2]]).all() and not torch.isnan(ref[off[2]:]).any()
    _near(got, ref, O.rounded(ref, bound, torch.bfloat16), "out")
    # a table that is too short for the lengths
    got = M.attend(q, cache, table[:, :3].contiguous(), lens, None if one else torch.tensor(off, dtype=torch.int32).cuda())
    ref, bound = O.attend(q, *cache, [r[:3] for r in rows], lengths, None if one else off)
    _near(got, ref, O.rounded(ref, bound, torch.bfloat16), "out")


@pytest.mark.gpu
@pytest.mark.parametrize("top", [2 ** 31 - 1, 5000])
@pytest.mark.parametrize("width,per", [(8, 1), (60, 1), (8, 2), (60, 40)])
def test_lengths_far_past_the_table(width, per, top):
    """A length that no table holds costs no more than the table: its rows are NaN, the other streams' what they are."""
    from robustvideomatting_amd import temporal as M
    g, dt, lengths = _gen(6), torch.float16, [20, 30, 3]
    cache, table, rows, lens = _attend_case(g, lengths, [per] * 3, 4, 2, 64, 16, dt, 0.0)
    wide = torch.full((3, width), 0, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    off = None if per == 1 else torch.tensor(_offsets([per] * 3), dtype=torch.int32).cuda()
    q, kv = _rn(g, 3 * per, 4, 64, dtype=dt), _rn(g, 3 * per, 2, 64, dtype=dt)
    clean = M.attend(q, cache, wide, lens, off)
    lens[1] = top
    keep = [c.clone() for c in cache]
    got = M.attend(q, cache, wide, lens, off)
    mine = slice(per, 2 * per)
    assert torch.isnan(got[mine]).all()
    got[mine] = clean[mine]
    assert torch.equal(got, clean)
    lens[0] = lens[2] = -100
    M.append_kv(kv, kv, cache, wide, lens, off)
    assert torch.equal(cache[0], keep[0]) and torch.equal(cache[1], keep[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("longest", [60, 2500])
def test_attend_many_streams_with_one_token(dtype, longest):
    """More streams than a wave has lanes, some without a token, two tiles of query heads, in both forms."""
    from robustvideomatting_amd import temporal as M
    dt, g, S = DT[dtype], _gen(longest), 150
    lengths = [(37 * i) % 61 - 8 for i in range(S)]
    lengths[97] = longest
    cache, table, rows, lens = _attend_case(g, lengths, [1] * S, 20, 1, 32, 16, dt, float("nan"))
    q = _rn(g, S, 20, 32, dtype=dt)
    got = M.attend(q, cache, table, lens)
    ref, bound = O.attend(q, *cache, rows, lengths, None)
    _near(got, ref, O.rounded(ref, bound, dt), "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_rows_before_the_first_stream(dtype):
    """Packed rows that begin and end with rows of no stream: they come out as 0 and store nothing."""
    from robustvideomatting_amd import temporal as M
    dt, g, lengths, off = DT[dtype], _gen(31), [5, 0, 100], [3, 10, 10, 45]
    cache, table, rows, lens = _attend_case(g, lengths, [7, 0, 35], 4, 2, 64, 16, dt, 0.0)
    offsets = torch.tensor(off, dtype=torch.int32).cuda()
    q, k = _rn(g, 50, 4, 64, dtype=dt), _rn(g, 50, 2, 64, dtype=dt)
    before = [c.clone() for c in cache]
    qr = M.append_kv(k, k, cache, table, lens, offsets, q=q)
    assert not qr[:3].any() and not qr[45:].any() and torch.equal(qr[3:45], q[3:45])
    changed = [(c != b).any(-1).any(1).sum().item() for c, b in zip(cache, before)]
    assert changed == [42, 42]
    got = M.attend(qr, cache, table, lens, offsets)
    ref, bound = O.attend(qr, *cache, rows, lengths, off)
    assert not got[:3].any() and not got[45:].any()
    _near(got, ref, O.rounded(ref, bound, dt), "out")


@pytest.mark.gpu
def test_frames_one_by_one_and_in_one_chunk():
    """A stream's clip appended and attended in one call, and frame by frame through a growing cache."""
    from robustvideomatting_amd import temporal as M
    g, dt, Hq, Hkv, Dh, page, T, per = _gen(2), torch.float16, 4, 2, 64, 16, 6, 7
    freqs = (10000.0 ** (-torch.arange(0, 64, 2).float() / 64)).cuda()
    S = 3
    q, k, v = (_rn(g, S, T * per, h, Dh, dtype=dt) for h in (Hq, Hkv, Hkv))
    new = [T * per] * S

    def fresh():
        cache, table, rows, lens = _paged(_gen(3), [0] * S, new, Hkv, Dh, page, dt)
        return cache, table, lens

    cache, table, lens = fresh()
    off = torch.tensor(_offsets(new), dtype=torch.int32).cuda()
    qr = M.append_kv(k.flatten(0, 1), v.flatten(0, 1), cache, table, lens, off, freqs=freqs, q=q.flatten(0, 1))
    whole = M.attend(qr, cache, table, lens, off).view(S, T * per, Hq, Dh)
    cache2, table2, lens2 = fresh()
    off2 = torch.tensor(_offsets([per] * S), dtype=torch.int32).cuda()
    for t in range(T):
        sl = slice(t * per, (t + 1) * per)
        qr = M.append_kv(k[:, sl].flatten(0, 1), v[:, sl].flatten(0, 1), cache2, table2, lens2, off2, freqs=freqs, q=q[:, sl].flatten(0, 1))
        part = M.attend(qr, cache2, table2, lens2, off2).view(S, per, Hq, Dh)
        # both are within half a step (and the weights' half steps) of the same value
        assert (part.double() - whole[:, sl].double()).abs().max() <= 4 * O.half_step(dt) * v.abs().max().item()
        lens2 += per
    assert torch.equal(cache[0], cache2[0]) and torch.equal(cache[1], cache2[1])


@pytest.mark.gpu
def test_pages_past_32_bits():
    """A pool of more than 2^32 elements: its last pages hold what a small pool would."""
    from robustvideomatting_amd import temporal as M
    g, dt, Hkv, page, Dh = _gen(12), torch.float16, 2, 1024, 128
    pages = (1 << 32) // (Hkv * page * Dh) + 40
    lengths, new = [1500, 7, 3000], [1, 40, 300]
    small, table, rows, lens = _attend_case(g, lengths, new, Hkv, Hkv, Dh, page, dt, 0.0)
    n = small[0].shape[0]
    big = tuple(torch.empty((pages, Hkv, page, Dh), dtype=dt, device="cuda") for _ in range(2))
    for b, s in zip(big, small):
        b[-n:] = s
    far = torch.where(table < n, table + (pages - n), torch.full_like(table, -1))
    assert big[0].numel() > 1 << 32
    for per in (1, 2):                                      # packed rows, and a row per stream
        off = torch.tensor(_offsets(new), dtype=torch.int32).cuda() if per == 1 else None
        R = sum(new) if per == 1 else len(new)
        q, k, v = (_rn(g, R, h, Dh, dtype=dt) for h in (4, Hkv, Hkv))
        freqs = (10000.0 ** (-torch.arange(0, Dh, 2).float() / Dh)).cuda()
        qs = M.append_kv(k, v, small, table, lens, off, freqs=freqs, q=q)
        qb = M.append_kv(k, v, big, far, lens, off, freqs=freqs, q=q)
        assert torch.equal(qs, qb) and torch.equal(big[0][-n:], small[0]) and torch.equal(big[1][-n:], small[1])
        assert torch.equal(M.attend(qb, big, far, lens, off), M.attend(qs, small, table, lens, off))


@pytest.mark.gpu
def test_sequences_past_32_bits():
    """Tensors of more than 2^31 elements: the last sequences are what they are alone."""
    from robustvideomatting_amd import temporal as M
    g, dt, B, T, D, N, last = _gen(13), torch.float16, 70000, 64, 512, 4, 1500
    x, step, A, Bm, Cm, Dv, bias = _scan_inputs(g, last, T, D, N, dt)
    w = _rn(g, 4, D, dtype=dt)
    big = torch.zeros((B, T, D), dtype=dt, device="cuda")
    assert big.numel() > 1 << 31
    big[-last:] = x
    y, state = M.causal_conv(big, w)
    ys, ss = M.causal_conv(x, w)
    assert torch.equal(y[-last:], ys) and torch.equal(state[-last:], ss)
    b, c = (torch.zeros((B, T, N), dtype=dt, device="cuda") for _ in range(2))
    b[-last:], c[-last:] = Bm, Cm
    y, h = M.selective_scan(big, big, A, b, c, Dv, big, bias)
    ys, hs = M.selective_scan(x, x, A, Bm, Cm, Dv, x, bias)
    assert torch.equal(y[-last:], ys) and torch.equal(h[-last:], hs)
    # one sequence: the tail continues from the state in front of it
    flat = big.view(1, B * T, D)
    y, _ = M.causal_conv(flat, w)
    ys, _ = M.causal_conv(flat[:, -1000:], w, state=flat[:, -1003:-1000])
    assert torch.equal(y[:, -1000:], ys)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_other_strides_and_orders(dtype):
    """Time-major, broadcast, channel-strided and unaligned inputs give the bits of dense ones, and dense results."""
    from robustvideomatting_amd import temporal as M
    dt, g = DT[dtype], _gen(14)
    B, T, D, N = 3, 70, 24, 16

    def forms(t):
        odd = torch.empty((*t.shape[:-1], 2 * t.shape[-1] + 1), dtype=t.dtype, device="cuda")
        odd[..., 1::2] = t
        return [t.transpose(0, 1).contiguous().transpose(0, 1), odd[..., 1::2], torch.cat([t[..., :1], t], -1)[..., 1:]]

    x, step, A, Bm, Cm, Dv, bias = _scan_inputs(g, B, T, D, N, dt)
    w, z = _rn(g, 4, D, dtype=dt), _rn(g, B, T, D, dtype=dt)
    c0, s0 = M.causal_conv(x, w)
    y0, h0 = M.selective_scan(x, step, A, Bm, Cm, Dv, z, bias)
    for xx, ss, bb, cc, zz in zip(*(forms(t) for t in (x, step, Bm, Cm, z))):
        c, s = M.causal_conv(xx, w.t().contiguous().t())
        y, h = M.selective_scan(xx, ss, A.t().contiguous().t(), bb, cc, Dv, zz, bias)
        assert torch.equal(c, c0) and torch.equal(s, s0) and torch.equal(y, y0) and torch.equal(h, h0)
        assert all(t.is_contiguous() for t in (c, s, y, h))
    one = [t[:1].expand(B, -1, -1) for t in (x, step, Bm, Cm, z)]       # the same sequence for all
    y, h = M.selective_scan(*one[:2], A, *one[2:4], Dv, one[4], bias)
    assert torch.equal(y, y0[:1].expand(B, -1, -1)) and torch.equal(h, h0[:1].expand(B, -1, -1))
    cache, table, rows, lens = _attend_case(g, [20, 40, 0], [30, 1, 9], 2, 2, 32, 16, dt, 0.0)
    off = torch.tensor([0, 30, 31, 40], dtype=torch.int32).cuda()
    q, k = _rn(g, 40, 4, 32, dtype=dt), _rn(g, 40, 2, 32, dtype=dt)
    freqs = (10000.0 ** (-torch.arange(0, 32, 2).float() / 32)).cuda()
    r0 = M.append_kv(k, k, cache, table, lens, off, freqs=freqs, q=q)
    o0, keep = M.attend(r0, cache, table, lens, off), [c.clone() for c in cache]
    for qq, kk in zip(forms(q), forms(k)):
        r = M.append_kv(kk, kk, cache, table, lens, off, freqs=torch.stack([freqs, freqs], 1)[:, 0], q=qq)
        assert torch.equal(r, r0) and all(torch.equal(a, b) for a, b in zip(cache, keep))
    for rr in forms(r0):
        o = M.attend(rr, cache, table, lens, off)
        assert torch.equal(o, o0) and o.is_contiguous()


# ---- how they are called ----------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_refusals_on_the_device():
    from robustvideomatting_amd import temporal as M
    x = torch.zeros((1, 2, 8), device="cuda")
    w = torch.zeros((4, 8), device="cuda")
    with pytest.raises(RuntimeError, match="float16"):
        M.causal_conv(x, w.half())
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        M.causal_conv(x.double(), w.double())
    with pytest.raises(RuntimeError, match="shape"):
        M.causal_conv(x, w[:, :4])
    with pytest.raises(RuntimeError, match="taps"):
        M.causal_conv(x, torch.zeros((5, 8), device="cuda"))
    with pytest.raises(RuntimeError, match="state has shape"):
        M.causal_conv(x, w, state=torch.zeros((1, 4, 8), device="cuda"))
    with pytest.raises(RuntimeError, match="inference only"):
        M.causal_conv(x.clone().requires_grad_(), w)
    with torch.no_grad():
        M.causal_conv(x.clone().requires_grad_(), w)
    A, bc = torch.zeros((4, 8), device="cuda"), torch.zeros((1, 2, 4), device="cuda")
    with pytest.raises(RuntimeError, match="must be on"):
        M.selective_scan(x, x, A.cpu(), bc, bc)
    with pytest.raises(RuntimeError, match="C has shape"):
        M.selective_scan(x, x, A, bc, bc[..., :3])
    with pytest.raises(RuntimeError, match="states"):
        M.selective_scan(x, x, torch.zeros((65, 8), device="cuda"), torch.zeros((1, 2, 65), device="cuda"), torch.zeros((1, 2, 65), device="cuda"))
    pages = torch.zeros((2, 1, 16, 16), device="cuda")
    t = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    k = torch.zeros((2, 1, 16), device="cuda")
    with pytest.raises(RuntimeError, match="one row"):
        M.append_kv(k[:1], k[:1], (pages, pages), t, t[:, 0].contiguous())
    with pytest.raises(RuntimeError, match="int32"):
        M.attend(k, (pages, pages), t.long(), t[:, 0].contiguous())
    with pytest.raises(RuntimeError, match="dense"):
        M.attend(k, (pages.expand(2, 2, 16, 16), pages.expand(2, 2, 16, 16)), t, t[:, 0].contiguous())
    with pytest.raises(native_error(), match="scale"):
        M.attend(k, (pages, pages), t, t[:, 0].contiguous(), scale=0.0)
    with pytest.raises(native_error(), match="page size"):
        M.attend(k, (pages[:, :, :8].contiguous(), pages[:, :, :8].contiguous()), t, t[:, 0].contiguous())
    with pytest.raises(native_error(), match="rotated"):
        M.append_kv(k, k, (pages, pages), t, t[:, 0].contiguous(), freqs=torch.zeros(4, device="cuda"))


@pytest.mark.gpu
def test_tangents_are_refused_on_the_device():
    """Each tensor argument of each operator in turn."""
    import torch.autograd.forward_ad as F
    from robustvideomatting_amd import temporal as M
    z = lambda *shape: torch.zeros(shape, device="cuda")
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
    conv = dict(x=z(1, 2, 8), weight=z(4, 8), bias=z(8), state=z(1, 3, 8))
    scan = dict(x=z(1, 2, 8), dt=z(1, 2, 8), A=z(4, 8), B=z(1, 2, 4), C=z(1, 2, 4), D=z(8), z=z(1, 2, 8), dt_bias=z(8), state=z(1, 4, 8))
    append = dict(k=z(2, 1, 16), v=z(2, 1, 16), kp=z(2, 1, 16, 16), vp=z(2, 1, 16, 16), freqs=z(8), q=z(2, 1, 16))
    attend = dict(q=z(2, 1, 16), kp=z(2, 1, 16, 16), vp=z(2, 1, 16, 16))
    paged = lambda f: lambda kp, vp, **a: f(cache=(kp, vp), table=torch.tensor([[0], [1]], dtype=torch.int32, device="cuda"), lengths=i(2), **a)
    for call, args in ((M.causal_conv, conv), (M.selective_scan, scan), (paged(M.append_kv), append), (paged(M.attend), attend)):
        call(**args)
        with F.dual_level():
            call(**args)
            for name in args:
                with pytest.raises(RuntimeError, match="carries a tangent"):
                    call(**dict(args, **{name: F.make_dual(args[name], torch.ones_like(args[name]))}))


def native_error():
    from robustvideomatting_amd import native
    return native.NativeError


@pytest.mark.gpu
def test_empty_calls():
    from robustvideomatting_amd import temporal as M
    y, s = M.causal_conv(torch.zeros((0, 3, 8), device="cuda"), torch.zeros((4, 8), device="cuda"))
    assert y.shape == (0, 3, 8) and s.shape == (0, 3, 8)
    y, s = M.selective_scan(torch.zeros((0, 3, 8), device="cuda"), torch.zeros((0, 3, 8), device="cuda"), torch.zeros((4, 8), device="cuda"),
                            torch.zeros((0, 3, 4), device="cuda"), torch.zeros((0, 3, 4), device="cuda"))
    assert y.shape == (0, 3, 8) and s.shape == (0, 4, 8)
    pages = torch.zeros((2, 1, 16, 16), device="cuda")
    none = torch.zeros((0, 1, 16), device="cuda")
    t, z1 = torch.zeros((0, 1), dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    assert M.append_kv(none, none, (pages, pages), t, z1, q=none).shape == (0, 1, 16)
    assert M.attend(none, (pages, pages), t, z1).shape == (0, 1, 16)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    t2 = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    assert M.attend(none, (pages, pages), t2, off[:2].contiguous(), off).shape == (0, 1, 16)


def _everything(M, s):
    """The operators in a row, as a layer of a temporal model uses them."""
    y, s["conv"] = M.causal_conv(s["x"], s["w"], state=s["conv"])
    y, s["h"] = M.selective_scan(y, s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["bias"], s["h"])
    n, H, d = s["S"] * s["per"], 4, 64
    q = M.append_kv(y.reshape(n, 6, d)[:, 4:5], y.reshape(n, 6, d)[:, 5:], s["cache"], s["table"], s["lens"], s["off"], freqs=s["freqs"],
                    q=y.reshape(n, 6, d)[:, :H])
    o = M.attend(q, s["cache"], s["table"], s["lens"], s["off"])
    s["lens"] += s["per"]
    return o


def _layer(seed, per, S=2, room=64):
    g, D, N = _gen(seed), 6 * 64, 16
    s = dict(S=S, per=per)
    s["x"], s["dt"], s["z"] = (_rn(g, S, per, D, dtype=torch.float16) for _ in range(3))
    s["B"], s["C"] = (_rn(g, S, per, N, dtype=torch.float16) for _ in range(2))
    s["w"], s["A"], s["D"], s["bias"] = _rn(g, 4, D, dtype=torch.float16), -_rn(g, N, D).abs(), _rn(g, D), _rn(g, D)
    s["conv"], s["h"] = _rn(g, S, 3, D, dtype=torch.float16), _rn(g, S, N, D)
    s["cache"], s["table"], _, s["lens"] = _paged(g, [0] * S, [room * per] * S, 1, 64, 16, torch.float16)
    s["off"] = torch.arange(S + 1, dtype=torch.int32).cuda() * per if per > 1 else None
    s["freqs"] = (10000.0 ** (-torch.arange(0, 64, 2).float() / 64)).cuda()
    return s


@pytest.mark.gpu
@pytest.mark.parametrize("per", [1, 5, 700])
def test_captured_graph_follows_the_growing_cache(per):
    """The whole layer in a HIP graph, replayed as the cache grows, with eager work between the replays."""
    from robustvideomatting_amd import temporal as M
    a, b = _layer(1, per, room=8), _layer(1, per, room=8)
    state = {}

    def step(s):
        o = _everything(M, s)
        state["conv"], state["h"] = s["conv"], s["h"]
        return o

    want = []
    for _ in range(6):
        want.append(step(a).clone())
    stream = torch.cuda.Stream()
    conv0, h0, lens0 = b["conv"], b["h"], b["lens"].clone()
    torch.cuda.synchronize()                                # the other stream takes over
    with torch.cuda.stream(stream):
        keep = [c.clone() for c in b["cache"]]
        _everything(M, b)                                   # warm up
        b["conv"], b["h"] = conv0, h0
        b["lens"].copy_(lens0)
        for c, k in zip(b["cache"], keep):
            c.copy_(k)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = _everything(M, b)
        conv0.copy_(b["conv"])
        h0.copy_(b["h"])
    for i in range(6):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        junk = _everything(M, _layer(7, 3))                 # eager work of the same kind between the replays
        assert torch.isfinite(junk.float()).all()
    assert torch.equal(b["lens"], a["lens"]) and torch.equal(b["cache"][0], a["cache"][0])


@pytest.mark.gpu
def test_two_streams_at_once_and_another_stream_than_the_default():
    from robustvideomatting_amd import temporal as M
    want = [_everything(M, _layer(i, p)) for i, p in ((11, 1), (12, 300))]
    torch.cuda.synchronize()
    layers = [_layer(i, p) for i, p in ((11, 1), (12, 300))]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            got[i] = _everything(M, layers[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
