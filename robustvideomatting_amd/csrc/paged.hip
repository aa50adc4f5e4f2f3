// Appending tokens to a paged key-value cache, keys (and queries) rotated by their position on the way.
#include "temporal.hpp"

namespace {

constexpr int APPEND_THREADS = 256, APPEND_MAX_ROT = 256;

// k' (a, b) = (a cos t - b sin t, a sin t + b cos t) with t = position x freqs[i], stored with v at the token's slot.  A block per
// token, whose pieces are then all in flight at once and whose turns are computed once for all heads.  Bound by memory: 21.6k
// tokens of 16 + 8 + 8 heads x 128 in bf16, 353 MB moved, take 60.7 us, 5.8 TB/s; 64 single tokens are a launch (3.4 us).
// Sums of products in fp32, rounded once to the cache's type.
// ONCE: what is written does not fit the caches anyway and is written past them
template <typename T, bool INTER, bool ONCE>
__global__ __launch_bounds__(APPEND_THREADS) void append_kv(AppendArgs a) {
    typedef typename Vec<T, 8>::type V8;
    __shared__ float2 turn[APPEND_MAX_ROT / 2];
    const int m = blockIdx.x, tid = threadIdx.x;
    const PagedArgs& p = a.p;
    int pos;
    const int s = __builtin_amdgcn_readfirstlane(paged_row(p, m, pos));
    const bool mine = s < p.S && pos >= 0;
    // angle = position x frequency, exact in 64 bits (24 + 31 bits), reduced to a fraction of a turn before it is rounded to
    // 32: a 32-bit product is off by 2^-24 of the angle, whole radians for positions in the millions
    for (int i = tid; i < a.rot / 2; i += APPEND_THREADS) {
        const double rev = (double)pos * (double)a.freqs[i] * 0.15915494309189535;
        const float fr = (float)(rev - __builtin_rint(rev));
        turn[i] = make_float2(cospif(2.f * fr), sinpif(2.f * fr));
    }
    __syncthreads();
    const int pg = mine ? paged_page(p, s, pos) : -1, Dh = p.Dh;
    const int nch = Dh >> 3, npair = a.rot >> 4;                // 16-byte pieces of a head; pairs of pieces that rotate together
    const int nq = a.q ? p.Hq : 0, items = INTER ? nch : nch - npair;
    const int64_t slot = pos & ((1 << p.page_shift) - 1);
    auto put = [](T* to, V8 v) { if (ONCE) __builtin_nontemporal_store(v, (V8*)to); else *(V8*)to = v; };
    for (int i = tid; i < (nq + p.Hkv) * items; i += APPEND_THREADS) {
        const int h = i / items, c = i - h * items;
        const T* src; T* dst;
        if (h < nq) {
            src = (const T*)a.q + m * a.q_sm + h * a.q_sh;
            dst = (T*)a.q_out + ((int64_t)m * p.Hq + h) * Dh;
        } else {
            if (pg < 0) continue;
            src = (const T*)a.k + m * a.k_sm + (h - nq) * a.k_sh;
            dst = (T*)a.k_pages + ((((int64_t)pg * p.Hkv + h - nq) << p.page_shift) + slot) * Dh;
        }
        if (INTER) {
            V8 v = *(const V8*)(src + c * 8);
            if (c < 2 * npair) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 t = turn[c * 4 + j];
                    const float x = (float)v[2 * j], y = (float)v[2 * j + 1];
                    v[2 * j] = (T)(x * t.x - y * t.y); v[2 * j + 1] = (T)(x * t.y + y * t.x);
                }
            }
            if (s >= p.S) v = V8{};                             // a row of no stream
            put(dst + c * 8, v);
        } else if (c < npair) {
            V8 u = *(const V8*)(src + c * 8), v = *(const V8*)(src + a.rot / 2 + c * 8);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 t = turn[c * 8 + j];
                const float x = (float)u[j], y = (float)v[j];
                u[j] = (T)(x * t.x - y * t.y); v[j] = (T)(x * t.y + y * t.x);
            }
            if (s >= p.S) u = v = V8{};
            put(dst + c * 8, u);
            put(dst + a.rot / 2 + c * 8, v);
        } else {
            V8 v = *(const V8*)(src + (c + npair) * 8);
            if (s >= p.S) v = V8{};
            put(dst + (c + npair) * 8, v);
        }
    }
    if (pg < 0) return;
    for (int i = tid; i < p.Hkv * nch; i += APPEND_THREADS) {
        const int h = i / nch, c = i - h * nch;
        put((T*)a.v_pages + ((((int64_t)pg * p.Hkv + h) << p.page_shift) + slot) * Dh + c * 8,
            *(const V8*)((const T*)a.v + m * a.v_sm + h * a.v_sh + c * 8));
    }
}

template <typename T, bool ONCE> void run_append(const AppendArgs& a, hipStream_t s) {
    if (a.interleaved) append_kv<T, true, ONCE><<<a.p.M, APPEND_THREADS, 0, s>>>(a);
    else append_kv<T, false, ONCE><<<a.p.M, APPEND_THREADS, 0, s>>>(a);
}
// 21.6k tokens of 16 + 8 + 8 heads x 128 in bf16, 177 MB written: 64.5 us through the caches, 61.8 us past them.  Up to 32 MB
// (the second-level caches together) what is appended may still be there when the attention reads it
template <typename T> void run_append(const AppendArgs& a, hipStream_t s) {
    const int64_t bytes = (int64_t)a.p.M * (2 * a.p.Hkv + (a.q ? a.p.Hq : 0)) * a.p.Dh * (int)sizeof(T);
    if (bytes > (32 << 20)) run_append<T, true>(a, s); else run_append<T, false>(a, s);
}

}  // namespace

void launch_append_kv(const AppendArgs& a, int elem, hipStream_t s) {
    if (elem == ELEM_F32) run_append<float>(a, s);
    else if (elem == ELEM_F16) run_append<f16>(a, s);
    else run_append<bfl>(a, s);
}
