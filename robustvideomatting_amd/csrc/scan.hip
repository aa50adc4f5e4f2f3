// Causal convolution over time and selective state space scan, for chunks of steps and for single steps.
#include "temporal.hpp"
#include "scan_index.hpp"
#include <algorithm>

namespace {

__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float rcp_hw(float v) { return __builtin_amdgcn_rcpf(v); }
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
// v * sigmoid(v); v_exp_f32 and v_rcp_f32 are good to one unit of the last place
__device__ __forceinline__ float silu_f(float v) { return v * rcp_hw(1.f + exp2_hw(-LOG2E * v)); }
// log(1 + e^v) = max(v, 0) + log1p(e^-|v|).  Step sizes are often 1e-3 and below, where log(1 + e) would keep three or four
// digits of e: w = 1 + e is rounded, and what the rounding took off e, at most half a unit of 1, is added back to log(w) (over w,
// to be exact: 1 where e is small, and the term below a unit of the sum where it is not)
__device__ __forceinline__ float softplus_f(float v) {
    const float e = exp2_hw(-LOG2E * fabsf(v)), w = 1.f + e;
    return fmaxf(v, 0.f) + fmaf(LN2, __builtin_amdgcn_logf(w), e - (w - 1.f));
}

// 4^x h + e: a state behind many steps at once.  Where they make it grow past what a factor holds, the state itself may still be in
// range, zero or tiny as it was: two factors of 2^127 at most take any normal number past the range
__device__ __forceinline__ float carried(float x, float h, float e) {
    const float f = exp2_hw(fminf(x, 127.f));
    return fmaf(f * h, f, e);
}

// ---- causal convolution: y[t] = act(bias + sum_w weight[w] xx[t + w]) with xx = the W-1 rows of the state, then x ----
// A thread has VEC channels (16 bytes where the rows allow it) of RUN steps, taken four at a time with the next four requested ahead: the chip then
// reads, computes and writes at the same time, where threads that request a whole run at once go through the three together.
// The W-1 rows before a run are read again by the run before it (out of L2).
// Bound by memory: 2 x 8160 steps x 960 channels in bf16, 63 MB, take 15.0 us, 4.2 TB/s (a large copy: 5.2).  A run requested
// whole: 18.5 us; runs of 16 or 32 steps: slower.  A single step (8 x 960) is a launch: 3.5 us of kernel.
template <typename T, int VEC, int RUN, bool PAST>
__global__ __launch_bounds__(256) void causal_conv(CausalConvArgs a) {
    typedef typename Vec<T, VEC>::type V;
    const unsigned dv_n = a.D / VEC, id = blockIdx.x * 256 + threadIdx.x, bi = id / dv_n;
    const int d = (int)(id - bi * dv_n) * VEC;
    const int64_t b = bi / (unsigned)a.runs;
    const int run = (int)(bi - (unsigned)b * a.runs);
    if (b >= a.B) return;
    const int W = a.W, t0 = run * RUN;
    const T* x = (const T*)a.x + b * a.x_sb + d;
    const T* st = a.state_in ? (const T*)a.state_in + b * (W - 1) * a.D + d : nullptr;
    auto row = [&](int t) -> V {                        // step t; the state's rows are steps -(W-1) .. -1
        if (t >= 0) return *(const V*)(x + (int64_t)t * a.x_st);
        if (st) return *(const V*)(st + (int64_t)(t + W - 1) * a.D);
        return V{};
    };
    constexpr int BT = RUN < 4 ? RUN : 4;
    V in[BT + 3], next[BT], wt[4], bias = {};
    auto rows = [&](V* to, int t) {
#pragma unroll
        for (int k = 0; k < BT; ++k) to[k] = t + k < a.T ? row(t + k) : V{};
    };
    rows(next, t0);
#pragma unroll
    for (int k = 0; k < 3; ++k) in[BT + k] = k >= 4 - W && t0 + k - 3 < a.T ? row(t0 + k - 3) : V{};
#pragma unroll
    for (int k = 0; k < 4; ++k)                         // right-aligned: tap k of a shorter filter sits at k + 4 - W
        wt[k] = k >= 4 - W ? *(const V*)((const T*)a.weight + (int64_t)(k - (4 - W)) * a.D + d) : V{};
    if (a.bias) bias = *(const V*)((const T*)a.bias + d);
    T* y = (T*)a.y + (b * a.T) * a.D + d;
#pragma unroll
    for (int c = 0; c < RUN; c += BT) {
#pragma unroll
        for (int k = 0; k < 3; ++k) in[k] = in[BT + k];
#pragma unroll
        for (int k = 0; k < BT; ++k) in[k + 3] = next[k];
        if (c + BT < RUN) rows(next, t0 + c + BT);
#pragma unroll
        for (int k = 0; k < BT; ++k)
            if (t0 + c + k < a.T) {
                V o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float s = (float)bias[j];
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        if (w >= 4 - W) s = fmaf((float)wt[w][j], (float)in[k + w][j], s);
                    o[j] = (T)(a.silu ? silu_f(s) : s);
                }
                V* to = (V*)(y + (int64_t)(t0 + c + k) * a.D);
                if (PAST) __builtin_nontemporal_store(o, to); else *to = o;
            }
    }
    if (run == a.runs - 1) {
        T* so = (T*)a.state_out + b * (W - 1) * a.D + d;
        for (int k = 0; k < W - 1; ++k) *(V*)(so + (int64_t)k * a.D) = row(a.T - (W - 1) + k);
    }
}

template <typename T, int VEC, int RUN, bool PAST> void run_conv_n(CausalConvArgs a, hipStream_t s) {
    a.runs = a.T > RUN ? (a.T + RUN - 1) / RUN : 1;
    const int64_t n = (int64_t)a.B * a.runs * (a.D / VEC);
    causal_conv<T, VEC, RUN, PAST><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a);
}
// Runs of 8 steps where there are as many, single steps otherwise (one each: 13.9 us against 11.5 at 360 x 412 x 64).  y goes past the
// caches, which hold the rows that are read twice: 11.2 against 12.8 us at 24 x 412 steps x 960 channels - but only as rows of
// whole cache lines and most of one, which nobody else adds to (1530 x 412 x 24, 48-byte rows: 35.5 us past them, 22.9 through).
template <typename T, int VEC> void run_conv(const CausalConvArgs& a, hipStream_t s) {
    constexpr bool WIDE = VEC * sizeof(T) == 16;
    const size_t row = a.D * sizeof(T);
    if (a.T < 8) run_conv_n<T, VEC, 1, false>(a, s);
    else if (WIDE && (row % 64 == 0 || row >= 96)) run_conv_n<T, VEC, 8, WIDE>(a, s);
    else run_conv_n<T, VEC, 8, false>(a, s);
}
template <typename T> void run_conv_v(const CausalConvArgs& a, int vec, hipStream_t s) {
    if constexpr (sizeof(T) == 2) if (vec == 8) { run_conv<T, 8>(a, s); return; }
    if (vec == 4) run_conv<T, 4>(a, s);
    else if (vec == 2) run_conv<T, 2>(a, s);
    else run_conv<T, 1>(a, s);
}

// ---- selective scan: h_t = exp(delta_t A) h_(t-1) + delta_t x_t B_t,  y_t = C_t h_t + D x_t, times silu(z_t) ----
// One lane per channel with its N states in registers, a wave per 64 channels; B_t and C_t are the same for all channels and
// come out of LDS as broadcasts (converted to fp32 once per wave and step, not once per channel).  The next steps' inputs are
// requested before the present ones are worked on.  Where there are half or fewer channels than lanes, a wave has those of PACK
// sequences, whose B and C lie side by side in LDS.
// Bound by instructions, the exponential costing two of the others (8 cycles a wave).  One sequence of 8160 steps x 960 channels x
// 16 states, bf16, with a gate: 31 + 42 us in the two passes, the vector pipes busy for 89 and 94 % of them; its bytes would take
// 12.  4080 sequences of 12 steps x 64 channels: 16.6 us, bytes 10.7.
// Where there are too few (sequence, 64 channels) pairs for the chip, the time axis is cut into chunks, a wave each, the waves
// of a block being neighbours.  ENDS computes each chunk's last state from a zero start and the sum of its step sizes, and
// composes them over the block (the decay over a chunk is exp(A sum delta), see carried): every chunk's first state within its block, and
// the block's last.  FROM composes the blocks in front of it, then runs its chunks from there.
enum ScanMode { SCAN_WHOLE, SCAN_ENDS, SCAN_FROM };
constexpr int SCAN_WAVES = 8;                           // waves of a block where the time axis is cut (16: two thirds slower at 1021 steps)
template <int MODE> constexpr int scan_waves() { return MODE == SCAN_WHOLE ? 2 : SCAN_WAVES; }
template <int PACK> struct Lane { typedef int64_t type; };      // a lane's place from the wave's scalar address: of its sequence, too
template <> struct Lane<1> { typedef unsigned type; };
template <int NP> constexpr int scan_occupancy() { return NP <= 16 ? 4 : NP <= 32 ? 3 : 2; }      // waves of a SIMD

template <typename T, int NP, int PACK, int MODE>
__global__ __launch_bounds__((64 * scan_waves<MODE>()), scan_occupancy<NP>()) void selective_scan(ScanArgs a) {
    constexpr bool ENDS = MODE == SCAN_ENDS;
    constexpr int TB = scan_batch(NP, PACK), NV = scan_values(NP, ENDS), LD = scan_loads(NP, PACK, ENDS), W = scan_waves<MODE>();
    constexpr int BC = LD * 64, TAB = NP * 64;
    constexpr int LDS = MODE == SCAN_ENDS ? (W * (TAB + 64) > W * 2 * BC ? W * (TAB + 64) : W * 2 * BC) : MODE == SCAN_FROM ? W * 2 * BC + TAB : W * 2 * BC;
    __shared__ __attribute__((aligned(16))) float lds[LDS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned unit = MODE == SCAN_WHOLE ? blockIdx.x * W + wave : blockIdx.x;
    const unsigned bq = unit / (unsigned)a.dtiles;
    const int dti = (int)(unit - bq * (unsigned)a.dtiles), ch = MODE == SCAN_WHOLE ? 0 : blockIdx.y * W + wave;
    const int64_t b0 = (int64_t)bq * PACK;                              // the wave's first sequence
    if (MODE == SCAN_WHOLE && b0 >= a.B) return;
    const int last = PACK == 1 ? 0 : (int)min((int64_t)PACK, a.B - b0) - 1;
    const int seq = PACK == 1 ? 0 : min(lane / a.nD, last);             // the lane's, from there (lanes behind the last are idle)
    const int64_t b = b0 + seq;
    const int d_own = dti * 64 + lane - seq * a.nD, d = min(d_own, a.nD - 1);
    const bool own = d_own < a.nD;
    const int t0 = MODE == SCAN_WHOLE ? 0 : scan_first_step(a.T, a.chunk_len, ch), t1 = MODE == SCAN_WHOLE ? a.T : scan_end_step(a.T, a.chunk_len, t0);
    // a wave's rows are at scalar addresses plus 4 bytes times the lane; B and C are dealt over the lanes, each with a pointer of its own
    const char* x = (const char*)((const T*)a.x + b0 * a.x_sb + (int64_t)t0 * a.x_st);
    const char* dt = (const char*)((const T*)a.dt + b0 * a.dt_sb + (int64_t)t0 * a.dt_st);
    const char* z = MODE != SCAN_ENDS && a.z ? (const char*)((const T*)a.z + b0 * a.z_sb + (int64_t)t0 * a.z_st) : nullptr;
    const T* Bm = (const T*)a.Bm + b0 * a.B_sb + (int64_t)t0 * a.B_st;
    const T* Cm = (const T*)a.Cm + b0 * a.C_sb + (int64_t)t0 * a.C_st;
    const unsigned off = d * (unsigned)sizeof(T);
    typedef typename Lane<PACK>::type lane_t;
    const lane_t x_off = off + (lane_t)seq * (a.x_sb * (int)sizeof(T)), dt_off = off + (lane_t)seq * (a.dt_sb * (int)sizeof(T)),
                 z_off = off + (lane_t)seq * (a.z_sb * (int)sizeof(T)), y_off = off + (lane_t)seq * ((int64_t)a.T * a.nD * (int)sizeof(T));
    const int64_t x_step = a.x_st * (int)sizeof(T), dt_step = a.dt_st * (int)sizeof(T), z_step = a.z_st * (int)sizeof(T);
    T xr[TB], dr[TB], zr[TB], br[LD];
    const T* bp[LD];
    int64_t b_inc[LD];
#pragma unroll
    for (int j = 0; j < LD; ++j) {
        const int e = j * 64 + lane, v = e % NV, n = min(v % NP, a.N - 1), q = min(e / NV % PACK, last);
        const int64_t st = v < NP ? a.B_st : a.C_st;
        bp[j] = (v < NP ? Bm + q * a.B_sb : Cm + q * a.C_sb) + scan_step_of(e, NP, PACK, ENDS) * st + n;
        b_inc[j] = TB * st;
    }
    auto at = [&](const char* row, lane_t o) -> T { return *(const T*)(row + o); };
    auto load = [&](int left) {                         // the next `left` steps (TB or fewer: the last one again)
        if (left >= TB) {
#pragma unroll
            for (int i = 0; i < TB; ++i) { xr[i] = at(x + i * x_step, x_off); dr[i] = at(dt + i * dt_step, dt_off); }
            if (z)
#pragma unroll
                for (int i = 0; i < TB; ++i) zr[i] = at(z + i * z_step, z_off);
#pragma unroll
            for (int j = 0; j < LD; ++j) { br[j] = *bp[j]; bp[j] += b_inc[j]; }
        } else {
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const int64_t k = min(i, left - 1);
                xr[i] = at(x + k * x_step, x_off); dr[i] = at(dt + k * dt_step, dt_off);
                if (z) zr[i] = at(z + k * z_step, z_off);
            }
#pragma unroll
            for (int j = 0; j < LD; ++j) {
                const int k = scan_step_of(j * 64 + lane, NP, PACK, ENDS);
                br[j] = k < left ? *bp[j] : (T)0.f;
            }
        }
        x += TB * x_step; dt += TB * dt_step;
        if (z) z += TB * z_step;
    };
    if (t0 < t1) load(t1 - t0);
    // ---- first states.  States past N: decay 1, input 0, start 0 - they stay 0
    float h[NP], A2[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) A2[n] = a.A[(int64_t)min(n, a.N - 1) * a.nD + d];
    const float* first = a.state_in ? a.state_in + b * a.N * a.nD : nullptr;
    const int64_t slot = (b * a.chunks + ch) * (int64_t)a.nD;           // of this chunk in carry and steps
    float steps = 0.f;
    if (MODE == SCAN_FROM) {
        // the block's first state: a thread takes (n, channel) pairs and composes the blocks in front, requested eight at a time
        float* H = lds + W * 2 * BC;
        const int64_t per = (int64_t)a.nD * (a.N + 1);
        const float* tot = a.totals + (b * gridDim.y) * per + d;        // per block: N rows of last states, a row of step sums
        constexpr int NB = (NP + W - 1) / W, U = 8;
        float hb[NB], A2n[NB];
        int64_t row[NB];
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            row[k] = (int64_t)min(wave + k * W, a.N - 1) * a.nD;
            A2n[k] = a.A[row[k] + d] * (0.5f * LOG2E);
            hb[k] = first ? first[row[k] + d] : 0.f;
        }
        for (int j0 = 0; j0 < (int)blockIdx.y; j0 += U) {
            float e[U][NB], st[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float* at = tot + min(j0 + u, (int)blockIdx.y - 1) * per;
                st[u] = at[(int64_t)a.N * a.nD];
#pragma unroll
                for (int k = 0; k < NB; ++k) e[u][k] = at[row[k]];
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j0 + u < (int)blockIdx.y)
#pragma unroll
                    for (int k = 0; k < NB; ++k) hb[k] = carried(st[u] * A2n[k], hb[k], e[u][k]);
        }
#pragma unroll
        for (int k = 0; k < NB; ++k)
            if (wave + k * W < NP) H[(wave + k * W) * 64 + lane] = hb[k];
        const float before = 0.5f * a.steps[slot + d];
#pragma unroll
        for (int n = 0; n < NP; ++n) h[n] = a.carry[slot * a.N + (int64_t)min(n, a.N - 1) * a.nD + d];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            A2[n] = n < a.N ? A2[n] * LOG2E : 0.f;
            h[n] = n < a.N ? carried(A2[n] * before, H[n * 64 + lane], h[n]) : 0.f;
        }
    } else {
        if (MODE == SCAN_WHOLE && first) {
#pragma unroll
            for (int n = 0; n < NP; ++n) h[n] = first[(int64_t)min(n, a.N - 1) * a.nD + d];
        } else {
#pragma unroll
            for (int n = 0; n < NP; ++n) h[n] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            A2[n] = n < a.N ? A2[n] * LOG2E : 0.f;
            h[n] = n < a.N ? h[n] : 0.f;
        }
    }
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.f, skip = a.D ? a.D[d] : 0.f;
    char* y = (char*)((T*)a.y + (b0 * a.T + t0) * a.nD);
    const int64_t y_step = (int64_t)a.nD * (int)sizeof(T);
    int buf = 0;
    for (int t = t0; t < t1; t += TB, buf ^= 1) {
        float* bc = lds + (wave * 2 + buf) * BC;
        float xv[TB], dv[TB], zv[TB];
#pragma unroll
        for (int i = 0; i < TB; ++i) { xv[i] = (float)xr[i]; dv[i] = (float)dr[i] + bias; if (MODE != SCAN_ENDS) zv[i] = z ? (float)zr[i] : 0.f; }
#pragma unroll
        for (int j = 0; j < LD; ++j) bc[j * 64 + lane] = (j * 64 + lane) % NP < a.N ? (float)br[j] : 0.f;
        if (t + TB < t1) load(t1 - t - TB);
        if (a.softplus)
#pragma unroll
            for (int i = 0; i < TB; ++i) dv[i] = softplus_f(dv[i]);
        auto step = [&](int i) {
            const float delta = dv[i], dx = delta * xv[i];
            float o = MODE == SCAN_ENDS ? 0.f : skip * xv[i];
            if (MODE == SCAN_ENDS) steps += delta;
#pragma unroll
            for (int n4 = 0; n4 < NP; n4 += 4) {
                const f32x4 bv = *(const f32x4*)(bc + (i * PACK + seq) * NV + n4);
                f32x4 cv;
                if (MODE != SCAN_ENDS) cv = *(const f32x4*)(bc + (i * PACK + seq) * NV + NP + n4);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    h[n4 + k] = fmaf(exp2_hw(delta * A2[n4 + k]), h[n4 + k], dx * bv[k]);
                    if (MODE != SCAN_ENDS) o = fmaf(h[n4 + k], cv[k], o);
                }
            }
            if (MODE != SCAN_ENDS) {
                if (z) o *= silu_f(zv[i]);
                if (own) *(T*)(y + i * y_step + y_off) = (T)o;
            }
        };
        if (t + TB <= t1) {
#pragma unroll
            for (int i = 0; i < TB; ++i) { step(i); __builtin_amdgcn_sched_barrier(0); }      // (steps side by side cost registers, i.e. waves)
        } else {
#pragma unroll
            for (int i = 0; i < TB; ++i)
                if (t + i < t1) step(i);
        }
        y += TB * y_step;
    }
    if (MODE == SCAN_ENDS) {
        float* S = lds + W * TAB;                       // (the B values are done with)
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NP; ++n) lds[wave * TAB + n * 64 + lane] = h[n];
        S[wave * 64 + lane] = steps;
        __syncthreads();
        float* tot = a.totals + (b * gridDim.y + blockIdx.y) * (int64_t)a.nD * (a.N + 1) + d;
        const int64_t slot0 = (b * a.chunks + blockIdx.y * W) * (int64_t)a.nD;
        for (int n = wave; n < a.N; n += W) {
            const float A2n = a.A[(int64_t)n * a.nD + d] * (0.5f * LOG2E);
            float hb = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (own) a.carry[(slot0 + (int64_t)w * a.nD) * a.N + (int64_t)n * a.nD + d] = hb;
                hb = carried(A2n * S[w * 64 + lane], hb, lds[w * TAB + n * 64 + lane]);
            }
            if (own) tot[(int64_t)n * a.nD] = hb;
        }
        float sum = 0.f;
        for (int w = 0; w < wave; ++w) sum += S[w * 64 + lane];
        if (own) a.steps[slot + d] = sum;
        if (own && wave == W - 1) tot[(int64_t)a.N * a.nD] = sum + steps;
        return;
    }
    if (!own || (MODE == SCAN_FROM && ch != a.chunks - 1)) return;
    float* out = a.state_out + b * a.N * a.nD;
#pragma unroll
    for (int n = 0; n < NP; ++n)
        if (n < a.N) out[(int64_t)n * a.nD + d] = h[n];
}

template <typename T, int NP, int PACK> void run_scan_n(const ScanArgs& a, hipStream_t s) {
    constexpr int W = SCAN_WAVES, WW = scan_waves<SCAN_WHOLE>();
    const unsigned units = (unsigned)((a.B + PACK - 1) / PACK * a.dtiles);
    if (a.chunks == 1) { selective_scan<T, NP, PACK, SCAN_WHOLE><<<(units + WW - 1) / WW, 64 * WW, 0, s>>>(a); return; }
    const dim3 grid(units, (unsigned)(a.chunks / W));
    selective_scan<T, NP, PACK, SCAN_ENDS><<<grid, 64 * W, 0, s>>>(a);
    selective_scan<T, NP, PACK, SCAN_FROM><<<grid, 64 * W, 0, s>>>(a);
}
template <typename T, int NP> void run_scan_p(const ScanArgs& a, int pack, hipStream_t s) {
    if constexpr (NP <= 16) if (pack == 4) { run_scan_n<T, NP, 4>(a, s); return; }
    if constexpr (NP <= 32) if (pack == 2) { run_scan_n<T, NP, 2>(a, s); return; }
    run_scan_n<T, NP, 1>(a, s);
}
template <typename T> void run_scan(const ScanArgs& a, int pack, hipStream_t s) {
    if (a.N <= 8) run_scan_p<T, 8>(a, pack, s);
    else if (a.N <= 16) run_scan_p<T, 16>(a, pack, s);
    else if (a.N <= 32) run_scan_p<T, 32>(a, pack, s);
    else run_scan_p<T, 64>(a, pack, s);
}

}  // namespace

// the widest pieces, of 16 bytes at most, that divide the channels and that every row starts on
void launch_causal_conv(const CausalConvArgs& a, int elem, hipStream_t s) {
    const int es = elem == ELEM_F32 ? 4 : 2;
    auto fits = [&](int vec) {
        auto on = [&](const void* p) { return (uintptr_t)p % (vec * es) == 0; };
        return a.D % vec == 0 && a.x_sb % vec == 0 && a.x_st % vec == 0 && on(a.x) && on(a.weight) && on(a.bias) && on(a.state_in) &&
               on(a.y) && on(a.state_out);
    };
    int vec = 16 / es;
    while (vec > 1 && !fits(vec)) vec /= 2;
    if (elem == ELEM_F32) run_conv_v<float>(a, vec, s);
    else if (elem == ELEM_F16) run_conv_v<f16>(a, vec, s);
    else run_conv_v<bfl>(a, vec, s);
}

// Chunks of the time axis, a multiple of a block's waves: none where every SIMD has a wave without them, otherwise as many as
// give it four waves (what the registers allow), of 8 steps at least, or 12 where there are two waves per SIMD even so (3 x 1021
// steps x 333, fp32: 29 us in 8, 25 in 12; 1 x 512 x 960, bf16: 18 and 21).  512 steps x 960 channels, bf16: 60 sequences 212 us in
// chunks and 247 without, 70 sequences 247 and 249, 100 sequences 307 and 255.  16 sequences of 32 steps 17 in chunks and 16
// without, of 48 steps 18 and 22; 40 of 63 steps 36 both ways.
constexpr int SCAN_MIN_STEPS = 8;
// Sequences of a wave: as many as its lanes hold (4 or 2: their B and C go through the same registers), where the chip has four
// waves per SIMD even with a sequence each.  1000 x 200 steps x 16 channels, bf16, 16 states: 36 us against 95 with one each;
// 667 x 575 x 26, 8 states: 89 against 123.
int scan_pack(int B, int T, int D, int N) {
    if (D > 32 || N > 32 || (T < 64 ? B : (int64_t)B * (T / SCAN_MIN_STEPS)) < 4096) return 1;
    return D <= 16 && N <= 16 ? 4 : 2;
}
int scan_chunks(int B, int T, int D, int N) {
    const int pack = scan_pack(B, T, D, N);
    const int64_t waves = ((int64_t)B + pack - 1) / pack * ((D + 63) / 64), W = SCAN_WAVES;
    if (waves >= 1024 || T < (waves > 512 ? 64 : 40)) return 1;
    const int64_t most = std::max(W, 4096 / waves / W * W), least = waves * (T / SCAN_MIN_STEPS) <= 2048 ? SCAN_MIN_STEPS : SCAN_MIN_STEPS + SCAN_BATCH;
    const int64_t len = std::max(least, scan_chunk_len(T, most));
    return (int)(((T + len - 1) / len + W - 1) / W * W);
}
int64_t scan_workspace_floats(int64_t B, int64_t chunks, int64_t D, int64_t N) {
    return B * (chunks + chunks / SCAN_WAVES) * (N + 1) * D;
}
void launch_selective_scan(const ScanArgs& a0, int elem, hipStream_t s) {
    ScanArgs a = a0;
    a.dtiles = (a.nD + 63) / 64;
    a.chunk_len = a.chunks > 1 ? (int)scan_chunk_len(a.T, a.chunks) : a.T;
    a.steps = a.carry + (int64_t)a.B * a.chunks * a.N * a.nD;
    a.totals = a.steps + (int64_t)a.B * a.chunks * a.nD;
    const int pack = scan_pack(a.B, a.T, a.nD, a.N);
    if (elem == ELEM_F32) run_scan<float>(a, pack, s);
    else if (elem == ELEM_F16) run_scan<f16>(a, pack, s);
    else run_scan<bfl>(a, pack, s);
}
