// Causal convolution over time and selective state space scan, for chunks of steps and for single steps.
#include "temporal.hpp"

namespace {

__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float rcp_hw(float v) { return __builtin_amdgcn_rcpf(v); }
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
// v * sigmoid(v); v_exp_f32 and v_rcp_f32 are good to one unit of the last place
__device__ __forceinline__ float silu_f(float v) { return v * rcp_hw(1.f + exp2_hw(-LOG2E * v)); }
// log(1 + e^v) = max(v, 0) + log1p(e^-|v|).  Step sizes are often 1e-3 and below, where log(1 + e) would keep three or four
// digits of e: w = 1 + e is rounded, and log(w) e / (w - 1) puts back what the rounding took (the quotient varies slowly)
__device__ __forceinline__ float softplus_f(float v) {
    const float e = exp2_hw(-LOG2E * fabsf(v)), w = 1.f + e, d = w - 1.f;
    const float lg = LN2 * __builtin_amdgcn_logf(w);
    return fmaxf(v, 0.f) + (d == 0.f ? e : lg * e * rcp_hw(d));
}

// ---- causal convolution: y[t] = act(bias + sum_w weight[w] xx[t + w]) with xx = the W-1 rows of the state, then x ----
constexpr int CONV_RUN = 16;                            // steps per thread: the W-1 rows before a run are read twice

template <typename T, int VEC>
__global__ __launch_bounds__(256) void causal_conv(CausalConvArgs a) {
    typedef typename Vec<T, VEC>::type V;
    const int dv_n = a.D / VEC;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t bi = id / dv_n;
    const int d = (int)(id - bi * dv_n) * VEC, run = (int)(bi % a.runs);
    const int64_t b = bi / a.runs;
    if (b >= a.B) return;
    const int W = a.W, t0 = run * CONV_RUN, t1 = min(a.T, t0 + CONV_RUN);
    const T* x = (const T*)a.x + b * a.x_sb + d;
    const T* st = a.state_in ? (const T*)a.state_in + b * (W - 1) * a.D + d : nullptr;
    auto row = [&](int i) -> V {                        // row i of xx
        if (i >= W - 1) return *(const V*)(x + (int64_t)(i - (W - 1)) * a.x_st);
        if (st) return *(const V*)(st + (int64_t)i * a.D);
        return V{};
    };
    float w[4][VEC], win[4][VEC], bias[VEC];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) { w[k][j] = 0.f; win[k][j] = 0.f; }
        if (k >= 4 - W) {                               // right-aligned: tap k of a shorter filter sits at k + 4 - W
            const V v = *(const V*)((const T*)a.weight + (int64_t)(k - (4 - W)) * a.D + d);
#pragma unroll
            for (int j = 0; j < VEC; ++j) w[k][j] = (float)v[j];
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) bias[j] = a.bias ? (float)((const T*)a.bias)[d + j] : 0.f;
#pragma unroll
    for (int k = 0; k < 3; ++k)
        if (k >= 4 - W) {
            const V v = row(t0 + k - (4 - W));
#pragma unroll
            for (int j = 0; j < VEC; ++j) win[k + 1][j] = (float)v[j];
        }
    T* y = (T*)a.y + (b * a.T) * a.D + d;
    for (int t = t0; t < t1; ++t) {
        const V v = *(const V*)(x + (int64_t)t * a.x_st);
        V o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            win[0][j] = win[1][j]; win[1][j] = win[2][j]; win[2][j] = win[3][j]; win[3][j] = (float)v[j];
            float s = bias[j];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k >= 4 - W) s = fmaf(w[k][j], win[k][j], s);
            o[j] = (T)(a.silu ? silu_f(s) : s);
        }
        *(V*)(y + (int64_t)t * a.D) = o;
    }
    if (run == a.runs - 1) {
        T* so = (T*)a.state_out + b * (W - 1) * a.D + d;
        for (int k = 0; k < W - 1; ++k) *(V*)(so + (int64_t)k * a.D) = row(a.T + k);
    }
}

template <typename T, int VEC> void run_conv(const CausalConvArgs& a, hipStream_t s) {
    const int64_t n = (int64_t)a.B * a.runs * (a.D / VEC);
    causal_conv<T, VEC><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a);
}

// ---- selective scan: h_t = exp(delta_t A) h_(t-1) + delta_t x_t B_t,  y_t = C_t h_t + D x_t, times silu(z_t) ----
// One lane per channel with its N states in registers, a wave per 64 channels; B_t and C_t are the same for all channels and
// come out of LDS as broadcasts (converted to fp32 once per wave and step, not once per channel).  The next steps' inputs are
// requested before the present ones are worked on.
// Where there are too few (sequence, 64 channels) pairs for the chip, the time axis is cut into chunks: ENDS computes each
// chunk's last state from a zero start and the sum of its step sizes, scan_carry composes them (the decay over a chunk is
// exp(A sum delta)) into every chunk's first state, and FROM runs the chunks from there.
enum ScanMode { SCAN_WHOLE, SCAN_ENDS, SCAN_FROM };
constexpr int SCAN_WAVES = 4;
template <int NP> constexpr int scan_batch() { return NP <= 16 ? 8 : 4; }

template <typename T, int NP, int MODE>
__global__ __launch_bounds__(64 * SCAN_WAVES) void selective_scan(ScanArgs a) {
    constexpr int TB = scan_batch<NP>(), NV = MODE == SCAN_ENDS ? NP : 2 * NP, LD = (TB * NV + 63) / 64;
    __shared__ __attribute__((aligned(16))) float bc_lds[SCAN_WAVES][2][LD * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t unit = (int64_t)blockIdx.x * SCAN_WAVES + wave;
    const int dti = (int)(unit % a.dtiles), ch = (int)(unit / a.dtiles % a.chunks);
    const int64_t b = unit / a.dtiles / a.chunks;
    if (b >= a.B) return;
    const int d_own = dti * 64 + lane, d = min(d_own, a.nD - 1);
    const bool own = d_own < a.nD;
    const int t0 = MODE == SCAN_WHOLE ? 0 : ch * a.chunk_len, t1 = MODE == SCAN_WHOLE ? a.T : min(a.T, t0 + a.chunk_len);
    const int64_t slot = (b * a.chunks + ch) * (int64_t)a.nD;
    float h[NP], A2[NP];
    const float* h0 = MODE == SCAN_WHOLE ? (a.state_in ? a.state_in + b * a.N * a.nD : nullptr) : MODE == SCAN_FROM ? a.carry + slot * a.N : nullptr;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        A2[n] = n < a.N ? a.A[(int64_t)n * a.nD + d] * LOG2E : 0.f;
        h[n] = n < a.N && h0 ? h0[(int64_t)n * a.nD + d] : 0.f;
    }
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.f, skip = a.D ? a.D[d] : 0.f;
    float steps = 0.f;
    const T* x = (const T*)a.x + b * a.x_sb + d;
    const T* dt = (const T*)a.dt + b * a.dt_sb + d;
    const T* z = a.z ? (const T*)a.z + b * a.z_sb + d : nullptr;
    const T* Bm = (const T*)a.Bm + b * a.B_sb;
    const T* Cm = (const T*)a.Cm + b * a.C_sb;
    T* y = (T*)a.y + b * a.T * a.nD + d;
    T xr[TB], dr[TB], zr[TB], br[LD];
    auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            const int64_t ti = min(t + i, t1 - 1);
            xr[i] = x[ti * a.x_st];
            dr[i] = dt[ti * a.dt_st];
            if (MODE != SCAN_ENDS && z) zr[i] = z[ti * a.z_st];
        }
#pragma unroll
        for (int j = 0; j < LD; ++j) {
            const int e = j * 64 + lane, v = e % NV, n = v % NP;
            const int64_t ti = min(t + e / NV, t1 - 1);
            br[j] = n < a.N ? (v < NP ? Bm[ti * a.B_st + n] : Cm[ti * a.C_st + n]) : (T)0.f;
        }
    };
    if (t0 < t1) load(t0);
    int buf = 0;
    for (int t = t0; t < t1; t += TB, buf ^= 1) {
        float* bc = bc_lds[wave][buf];
        float xv[TB], dv[TB], zv[TB];
#pragma unroll
        for (int i = 0; i < TB; ++i) { xv[i] = (float)xr[i]; dv[i] = (float)dr[i] + bias; if (MODE != SCAN_ENDS && z) zv[i] = (float)zr[i]; }
#pragma unroll
        for (int j = 0; j < LD; ++j) bc[j * 64 + lane] = (float)br[j];
        if (t + TB < t1) load(t + TB);
#pragma unroll
        for (int i = 0; i < TB; ++i)
            if (t + i < t1) {
                const float delta = a.softplus ? softplus_f(dv[i]) : dv[i], dx = delta * xv[i];
                float o = MODE == SCAN_ENDS ? 0.f : skip * xv[i];
                if (MODE == SCAN_ENDS) steps += delta;
#pragma unroll
                for (int n4 = 0; n4 < NP; n4 += 4) {
                    const f32x4 bv = *(const f32x4*)(bc + i * NV + n4);
                    f32x4 cv;
                    if (MODE != SCAN_ENDS) cv = *(const f32x4*)(bc + i * NV + NP + n4);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        h[n4 + k] = fmaf(exp2_hw(delta * A2[n4 + k]), h[n4 + k], dx * bv[k]);
                        if (MODE != SCAN_ENDS) o = fmaf(h[n4 + k], cv[k], o);
                    }
                }
                if (MODE != SCAN_ENDS) {
                    if (z) o *= silu_f(zv[i]);
                    if (own) y[(int64_t)(t + i) * a.nD] = (T)o;
                }
            }
    }
    if (!own || MODE == SCAN_FROM) return;
    float* out = MODE == SCAN_WHOLE ? a.state_out + b * a.N * a.nD : a.carry + slot * a.N;
#pragma unroll
    for (int n = 0; n < NP; ++n)
        if (n < a.N) out[(int64_t)n * a.nD + d] = h[n];
    if (MODE == SCAN_ENDS) a.steps[slot + d] = steps;
}

// every chunk's first state in place of its last one, and the sequence's last state
__global__ __launch_bounds__(256) void scan_carry(ScanArgs a) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (int64_t)a.N * a.nD, b = id / per;
    if (b >= a.B) return;
    const int64_t nd = id - b * per;
    const int d = (int)(nd % a.nD);
    const float A2 = a.A[nd] * LOG2E;
    float h = a.state_in ? a.state_in[id] : 0.f;
    float* c = a.carry + b * a.chunks * per + nd;
    const float* st = a.steps + b * a.chunks * a.nD + d;
    constexpr int U = 8;
    for (int i = 0; i < a.chunks; i += U) {
        float e[U], s[U];
#pragma unroll
        for (int k = 0; k < U; ++k) { const int64_t j = min(i + k, a.chunks - 1); e[k] = c[j * per]; s[k] = st[j * a.nD]; }
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (i + k < a.chunks) { c[(i + k) * per] = h; h = fmaf(exp2_hw(s[k] * A2), h, e[k]); }
    }
    a.state_out[id] = h;
}

template <typename T, int NP> void run_scan_n(const ScanArgs& a, hipStream_t s) {
    const int64_t units = (int64_t)a.B * a.dtiles * a.chunks;
    const unsigned g = (unsigned)((units + SCAN_WAVES - 1) / SCAN_WAVES);
    if (a.chunks == 1) { selective_scan<T, NP, SCAN_WHOLE><<<g, 64 * SCAN_WAVES, 0, s>>>(a); return; }
    selective_scan<T, NP, SCAN_ENDS><<<g, 64 * SCAN_WAVES, 0, s>>>(a);
    scan_carry<<<(unsigned)(((int64_t)a.B * a.N * a.nD + 255) / 256), 256, 0, s>>>(a);
    selective_scan<T, NP, SCAN_FROM><<<g, 64 * SCAN_WAVES, 0, s>>>(a);
}
template <typename T> void run_scan(const ScanArgs& a, hipStream_t s) {
    if (a.N <= 8) run_scan_n<T, 8>(a, s);
    else if (a.N <= 16) run_scan_n<T, 16>(a, s);
    else if (a.N <= 32) run_scan_n<T, 32>(a, s);
    else run_scan_n<T, 64>(a, s);
}

}  // namespace

void launch_causal_conv(const CausalConvArgs& a0, int elem, hipStream_t s) {
    CausalConvArgs a = a0;
    a.runs = a.T > 0 ? (a.T + CONV_RUN - 1) / CONV_RUN : 1;
    const size_t es = elem == ELEM_F32 ? 4 : 2;
    const int vec = 16 / (int)es;
    auto ok = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
    const bool wide = a.D % vec == 0 && a.x_sb % vec == 0 && a.x_st % vec == 0 && ok(a.x) && ok(a.weight) && ok(a.state_in) &&
                      ok(a.y) && ok(a.state_out);
    if (elem == ELEM_F32) { if (wide) run_conv<float, 4>(a, s); else run_conv<float, 1>(a, s); }
    else if (elem == ELEM_F16) { if (wide) run_conv<f16, 8>(a, s); else run_conv<f16, 1>(a, s); }
    else { if (wide) run_conv<bfl, 8>(a, s); else run_conv<bfl, 1>(a, s); }
}

// Chunks of the time axis: none where every SIMD has a wave without them, otherwise as many as give it four, of 32 steps at least
int scan_chunks(int B, int T, int D) {
    const int64_t waves = (int64_t)B * ((D + 63) / 64);
    if (waves >= 1024 || T < 64) return 1;
    int64_t n = (4096 + waves - 1) / waves;
    if (n > T / 32) n = T / 32;
    const int len = (int)((T + n - 1) / n + 7) / 8 * 8;
    return (T + len - 1) / len;
}
void launch_selective_scan(const ScanArgs& a0, int elem, hipStream_t s) {
    ScanArgs a = a0;
    a.dtiles = (a.nD + 63) / 64;
    a.chunk_len = a.chunks > 1 ? ((a.T + a.chunks - 1) / a.chunks + 7) / 8 * 8 : a.T;
    if (elem == ELEM_F32) run_scan<float>(a, s);
    else if (elem == ELEM_F16) run_scan<f16>(a, s);
    else run_scan<bfl>(a, s);
}
