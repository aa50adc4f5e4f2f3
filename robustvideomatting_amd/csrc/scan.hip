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
// One lane per channel with its N states in registers.
template <typename T, int NP>
__global__ __launch_bounds__(64) void selective_scan(ScanArgs a) {
    const int lane = threadIdx.x;
    const int dt_i = blockIdx.x % a.dtiles;
    const int64_t b = blockIdx.x / a.dtiles;
    const int d_own = dt_i * 64 + lane, d = min(d_own, a.nD - 1);
    const bool own = d_own < a.nD;
    float h[NP], A2[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        A2[n] = n < a.N ? a.A[(int64_t)n * a.nD + d] * LOG2E : 0.f;
        h[n] = n < a.N && a.state_in ? a.state_in[(b * a.N + n) * a.nD + d] : 0.f;
    }
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.f, skip = a.D ? a.D[d] : 0.f;
    const T* x = (const T*)a.x + b * a.x_sb + d;
    const T* dt = (const T*)a.dt + b * a.dt_sb + d;
    const T* z = a.z ? (const T*)a.z + b * a.z_sb + d : nullptr;
    const T* Bm = (const T*)a.Bm + b * a.B_sb;
    const T* Cm = (const T*)a.Cm + b * a.C_sb;
    T* y = (T*)a.y + b * a.T * a.nD + d;
    for (int64_t t = 0; t < a.T; ++t) {
        const float xv = (float)x[t * a.x_st], raw = (float)dt[t * a.dt_st] + bias;
        const float delta = a.softplus ? softplus_f(raw) : raw, dx = delta * xv;
        float o = skip * xv;
#pragma unroll
        for (int n = 0; n < NP; ++n)
            if (n < a.N) {
                h[n] = fmaf(exp2_hw(delta * A2[n]), h[n], dx * (float)Bm[t * a.B_st + n]);
                o = fmaf(h[n], (float)Cm[t * a.C_st + n], o);
            }
        if (z) o *= silu_f((float)z[t * a.z_st]);
        if (own) y[t * a.nD] = (T)o;
    }
    if (own)
#pragma unroll
        for (int n = 0; n < NP; ++n)
            if (n < a.N) a.state_out[(b * a.N + n) * a.nD + d] = h[n];
}

template <typename T> void run_scan(const ScanArgs& a, hipStream_t s) {
    const unsigned g = (unsigned)(a.B * a.dtiles);
    if (a.N <= 8) selective_scan<T, 8><<<g, 64, 0, s>>>(a);
    else if (a.N <= 16) selective_scan<T, 16><<<g, 64, 0, s>>>(a);
    else if (a.N <= 32) selective_scan<T, 32><<<g, 64, 0, s>>>(a);
    else selective_scan<T, 64><<<g, 64, 0, s>>>(a);
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

int scan_chunks(int, int, int) { return 1; }
void launch_selective_scan(const ScanArgs& a0, int elem, hipStream_t s) {
    ScanArgs a = a0;
    a.dtiles = (a.nD + 63) / 64;
    if (elem == ELEM_F32) run_scan<float>(a, s);
    else if (elem == ELEM_F16) run_scan<f16>(a, s);
    else run_scan<bfl>(a, s);
}
