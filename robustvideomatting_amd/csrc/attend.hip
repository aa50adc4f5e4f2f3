// Attention of new tokens over a paged key-value cache: softmax_j(scale q . k_j) v_j, one pass over the cache with a running
// maximum and sum.  Both kernels compute the transposed products
//     S' = K Q'   (keys x rows)        O' = V' P'   (dims x rows)
// because the accumulator of the first then holds, per lane, scores of ONE row: its maximum and sum are in-lane but for one or
// two exchanges, the rescale of O' is a lane's own, and the weights P' are the B operand of the second product where they
// stand - the matrix instruction sums over its K slots in any order, so V' is simply read in the order the scores came out.
//   attend_one    one new token per stream: the rows of a tile are the query heads that share a key head (16 x 16 tiles)
//   attend_chunk  many rows per stream: (token, head of the group) pairs share every key they read (32 x 32 tiles)
#include "temporal.hpp"
#include <algorithm>
#include <atomic>
#include <type_traits>

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef Vec<bfl, 8>::type b16x8;

__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }

// ---- a tile of keys or values in LDS: rows of DP elements in 16-byte pieces, the pieces of a row permuted by XOR so that the
// reads below spread over all banks (64 banks of 4 bytes: 16 pieces side by side; RPL rows of a narrow tile share a line)
template <typename T, int DP> struct Tile {
    static constexpr int PER = 16 / (int)sizeof(T), CPR = DP / PER, RPL = CPR >= 16 ? 1 : 16 / CPR, PITCH = DP * (int)sizeof(T);
    // keys: 16 rows, the same piece of each
    __device__ static __forceinline__ int kswz(int row, int c) { return c ^ ((row / RPL) & (CPR < 16 ? CPR - 1 : 15)); }
    // values, 16-bit (transposing read, 32 lanes at a time): 8 rows, the same two pieces of each (MF = 16 x 16 tiles), or
    // 4 rows, the same four pieces (MF = 32); fp32: rows 4 apart, the same four (or eight)
    template <int MF> __device__ static __forceinline__ int vswz(int row, int c) {
        if constexpr (sizeof(T) == 2) return c ^ (((row / RPL) << (MF == 16 ? 1 : 2)) & (CPR < 16 ? CPR - 1 : 15));
        else return c ^ ((((row >> 2) & 3) << 2) & (CPR - 1));
    }
    __device__ static __forceinline__ int koff(int row, int c) { return row * PITCH + kswz(row, c) * 16; }
    template <int MF> __device__ static __forceinline__ int voff(int row, int c) { return row * PITCH + vswz<MF>(row, c) * 16; }
};
// four rows x 16 columns of 16-bit elements, transposed: lane i of 16 gets column i of rows 0..3; the address of lane i is
// that of row i / 4, columns 4 (i % 4) ..
__device__ __forceinline__ s16x4 read_tr(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

__device__ __forceinline__ f32x4 mma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(b16x8 a, b16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(b16x8 a, b16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

template <typename V> __device__ __forceinline__ V as(u32x4 v) { return __builtin_bit_cast(V, v); }
// What is not there is read from here: a choice of addresses instead of a branch per load, behind which the compiler loses
// count of the loads in flight and waits for all of them.  (Global pointers, said so: a generic one counts as an LDS access.)
__device__ const u32x4 zero_piece = {0, 0, 0, 0};
typedef const __attribute__((address_space(1))) u32x4* GlobalPiece;
template <typename T> __device__ __forceinline__ u32x4 piece(const T* p, bool ok) {
    return *(ok ? (GlobalPiece)(uintptr_t)p : (GlobalPiece)(uintptr_t)&zero_piece);
}
// the same for what one block alone reads, once: not to be kept by the caches
template <typename T> __device__ __forceinline__ u32x4 piece_once(const T* p, bool ok) {
    return __builtin_nontemporal_load(ok ? (GlobalPiece)(uintptr_t)p : (GlobalPiece)(uintptr_t)&zero_piece);
}

// The matrix instruction takes weights of the tensors' type.  Each goes as two of them: rounded to it, and what that left out,
// so that 2 x 8 or 2 x 11 digits of it count.
template <typename T> struct TwoParts {
    typedef typename Vec<T, 8>::type V8;
    V8 upper, rest;
    __device__ __forceinline__ void set(int i, float w) { upper[i] = (T)w; rest[i] = (T)(w - (float)upper[i]); }
};
// Whether some of the pieces hold an infinity or NaN: times 0 it is not 0.  (Times a remainder, which has any sign or is 0, an infinite
// value is not what it is times the weight.)
__device__ __forceinline__ float times0(f16 a, f16 b, float s) { typedef Vec<f16, 2>::type V2; return __builtin_amdgcn_fdot2(V2{a, b}, V2{0, 0}, s, false); }
__device__ __forceinline__ float times0(bfl a, bfl b, float s) { typedef Vec<bfl, 2>::type V2; return __builtin_amdgcn_fdot2_f32_bf16(V2{a, b}, V2{0, 0}, s, false); }
template <typename T, int N> __device__ __forceinline__ bool any_not_finite(const u32x4 (&v)[N]) {
    float s[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const auto x = __builtin_bit_cast(typename Vec<T, 8>::type, v[j]);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] = times0(x[2 * k], x[2 * k + 1], s[k]);
    }
    return !((s[0] + s[1]) + (s[2] + s[3]) == 0.f);
}
template <typename V8> __device__ __forceinline__ V8 finite_only(V8 v) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (!__builtin_isfinite((float)v[k])) v[k] = 0;
    return v;
}

// ---- one token per stream -------------------------------------------------------------------------------------------------
// Work is cut by keys, not by streams: all streams' caches in units of NW tiles laid end to end, and block b of the grid
// takes the b-th equal share, whatever the streams' lengths - they are known on the device only.  A (stream, key head, 16 query
// heads) segment that fits inside a share is finished there; the pieces of one that does not go to the workspace (a block
// has at most two such pieces: its first and its last) and attend_join adds them up in order.
// Bound by memory: 8 streams of 8 to 65 thousand tokens, 8 key heads x 128 in bf16, 1.08 GB, take 178 us and 7 of joining, 6.1 TB/s
// (a large copy reads and writes 5.2).  Keys and values are read past the caches: 20 us more through them.  Weights in two parts cost
// nothing beside the loads, looking for infinities 3 % (256 dims: 7).  fp32, 1.85 GB: 298 us.  With rounded weights the result is off by 2.2e-3 of its size
// instead of the 1.7e-3 that one rounding to bf16 is (fp16: 2.5e-4, 2.1e-4).
template <typename T> constexpr int one_kt() { return sizeof(T) == 2 ? 32 : 16; }         // keys per tile of a wave
template <int DP> constexpr int one_nw() { return DP > 128 ? 2 : 4; }                      // waves of a block
// fp16 weights are taken times 2^14, which the quotient does not see: below 2^-14 the type loses digits
template <typename T> constexpr float one_lift() { return std::is_same<T, f16>::value ? 14.f : 0.f; }
constexpr int ONE_ROWS = 16, ONE_GRID = 512;
constexpr int piece_floats(int DP) { return ONE_ROWS * (DP + 2); }

// Where unit u of all units lies.  Run by a whole wave; uniform results.
struct Units {
    int64_t total, per;                 // units in all, of a block's share
    int stream, units;                  // stream of the unit asked for, units of each of its segments
    int64_t first;                      // first unit of that stream
    __device__ __forceinline__ static int of_stream(const PagedArgs& p, int s, int keys) {
        const int pos = s < p.S ? p.lengths[s] : -1;
        return pos < 0 ? 0 : (int)((paged_keys(p.width, p.page_shift, pos) - 1) / keys) + 1;
    }
    __device__ __forceinline__ void sum(const PagedArgs& p, int keys, int segs) {
        int64_t t = 0;
        for (int b = 0; b < p.S; b += 64) t += of_stream(p, b + (threadIdx.x & 63), keys);
        for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o);
        total = t * segs;
        per = (total + ONE_GRID - 1) / ONE_GRID;
    }
    // sets stream, units, first for unit u (0 <= u < total)
    __device__ __forceinline__ void find(const PagedArgs& p, int keys, int segs, int64_t u) {
        int64_t before = 0;
        const int lane = threadIdx.x & 63;
        for (int b = 0; b < p.S; b += 64) {
            const int mine = of_stream(p, b + lane, keys);
            int64_t inc = (int64_t)mine * segs;
            for (int o = 1; o < 64; o <<= 1) { const int64_t v = __shfl_up(inc, o); if (lane >= o) inc += v; }
            const unsigned long long hit = __ballot(before + inc > u);
            if (hit) {
                const int l = __ffsll(hit) - 1;
                stream = b + l;
                units = __shfl(mine, l);
                first = before + __shfl(inc, l) - (int64_t)units * segs;
                return;
            }
            before += __shfl(inc, 63);
        }
        stream = -1; units = 1; first = 0;
    }
};

template <typename T, int DP>
__global__ __launch_bounds__(64 * one_nw<DP>(), DP > 128 ? 1 : 2) void attend_one(AttendArgs a) {
    constexpr int NW = one_nw<DP>(), KT = one_kt<T>(), KEYS = NW * KT;
    typedef Tile<T, DP> TL;
    constexpr int LD = KT * TL::CPR / 64;                       // 16-byte pieces per lane of a K (or V) tile
    constexpr int DT = DP / 16, TILE_BYTES = KT * TL::PITCH;
    __shared__ __attribute__((aligned(16))) char lds[NW * 2 * TILE_BYTES];
    __shared__ float red_m[NW][16], red_l[NW][16];
    const PagedArgs& p = a.p;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    const int group = p.Hq / p.Hkv, rts = (group + 15) / 16, segs = p.Hkv * rts, Dh = p.Dh;
    char* kt_lds = lds + wave * 2 * TILE_BYTES;
    char* vt_lds = kt_lds + TILE_BYTES;

    // a stream without tokens has no unit: its row is 0
    auto clear = [&](int s, int h0, int h1) {
        for (int i = h0 * Dh + tid; i < h1 * Dh; i += 64 * NW) ((T*)a.out)[(int64_t)s * p.Hq * Dh + i] = (T)0.f;
    };
    Units U;
    int64_t u0, u1;
    if (a.splits) {
        U.sum(p, KEYS, segs);
        u0 = blockIdx.x * U.per; u1 = min(U.total, u0 + U.per);
        for (int s = blockIdx.x; s < p.S; s += gridDim.x)
            if (p.lengths[s] < 0) clear(s, 0, p.Hq);
    } else {                                                    // a block per segment, no pieces
        U.stream = blockIdx.x / segs; U.first = 0; U.units = Units::of_stream(p, U.stream, KEYS);
        const int seg = blockIdx.x - U.stream * segs;
        u0 = (int64_t)seg * U.units; u1 = u0 + U.units;
        if (!U.units && seg == 0) clear(U.stream, 0, p.Hq);
    }
    while (u0 < u1) {
        if (a.splits) U.find(p, KEYS, segs, u0);
        const int s = __builtin_amdgcn_readfirstlane(U.stream), n_units = __builtin_amdgcn_readfirstlane(U.units);
        const int seg = (int)((u0 - U.first) / n_units);
        const int64_t seg0 = U.first + (int64_t)seg * n_units;
        const int ua = (int)(u0 - seg0), ub = (int)min((int64_t)n_units, u1 - seg0);        // units of the segment done here
        const int kvh = seg / rts, h0 = kvh * group + (seg - kvh * rts) * 16, rows = min(16, kvh * group + group - h0);
        const int pos = p.lengths[s];
        const int t_end = ub * NW;                              // tiles, interleaved over the waves
        // ---- Q fragments: lane l15 is the row
        f32x4 acc[DT];
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[i] = f32x4{0, 0, 0, 0};
        u32x4 qf[TL::CPR / 4];
        const T* q = (const T*)a.q + s * a.q_sm + (h0 + min(l15, rows - 1)) * a.q_sh;
#pragma unroll
        for (int i = 0; i < TL::CPR / 4; ++i) qf[i] = piece(q + (4 * i + g) * TL::PER, (4 * i + g) * TL::PER < Dh);
        float m = -INFINITY, l = 0.f;
        bool lost = false;
        u32x4 kr[LD], vr[LD];
        // page numbers of a tile's groups of 16 keys, looked up a tile before they are used and by vector loads (each lane a
        // key of the group): a scalar load would be waited for together with the LDS reads
        int entry[KT / 16];
        const int* table = p.table + (int64_t)s * p.width;
        const int page_mask = (1 << p.page_shift) - 1;
        auto look = [&](int t) {
#pragma unroll
            for (int k = 0; k < KT / 16; ++k) entry[k] = table[min(((unsigned)t * KT + k * 16 + l15) >> p.page_shift, (unsigned)p.width - 1)];
        };
        auto load = [&](int t) {
#pragma unroll
            for (int j = 0; j < LD; ++j) {
                const int i = j * 64 + lane, row = i / TL::CPR, pc = i % TL::CPR, page = entry[KT > 16 ? j * 64 / TL::CPR >> 4 : 0];
                const unsigned key = (unsigned)t * KT + row;
                const bool here = (unsigned)page < (unsigned)p.pages && key >> p.page_shift < (unsigned)p.width, ok = here && key <= (unsigned)pos;
                lost |= !here && key <= (unsigned)pos;
                const int64_t base = ((((int64_t)page * p.Hkv + kvh) << p.page_shift) + (key & page_mask)) * Dh;
                const int kc = TL::kswz(row, pc) * TL::PER, vc = TL::template vswz<16>(row, pc) * TL::PER;
                kr[j] = piece_once((const T*)a.k_pages + base + kc, ok && kc < Dh);
                vr[j] = piece_once((const T*)a.v_pages + base + vc, ok && vc < Dh);
            }
        };
        int t = ua * NW + wave;
        if (t < t_end) { look(t); load(t); look(t + NW); }
        for (; t < t_end; t += NW) {
#pragma unroll
            for (int j = 0; j < LD; ++j) {
                *(u32x4*)(kt_lds + (j * 64 + lane) * 16) = kr[j];
                *(u32x4*)(vt_lds + (j * 64 + lane) * 16) = vr[j];
            }
            bool odd = false;
            if constexpr (sizeof(T) == 2) odd = __any(any_not_finite<T>(vr));
            if (t + NW < t_end) { load(t + NW); look(t + 2 * NW); }
            // ---- scores: lane = (row l15, keys 4 g .. 4 g + 3 of each 16)
            f32x4 sc[KT / 16];
#pragma unroll
            for (int kt = 0; kt < KT / 16; ++kt) {
                sc[kt] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < TL::CPR / 4; ++i) {
                    const u32x4 kf = *(const u32x4*)(kt_lds + TL::koff(kt * 16 + l15, 4 * i + g));
                    if constexpr (sizeof(T) == 2) sc[kt] = mma16(as<typename Vec<T, 8>::type>(kf), as<typename Vec<T, 8>::type>(qf[i]), sc[kt]);
                    else
#pragma unroll
                        for (int c = 0; c < 4; ++c) sc[kt] = mma16(as<f32x4>(kf)[c], as<f32x4>(qf[i])[c], sc[kt]);
                }
            }
            float mt = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < KT / 16; ++kt)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float v = sc[kt][c] * a.scale_log2e;
                    sc[kt][c] = kt * 16 + 4 * g + c <= pos - t * KT ? v : -INFINITY;
                    mt = fmaxf(mt, sc[kt][c]);
                }
            mt = fmaxf(mt, __shfl_xor(mt, 16));
            mt = fmaxf(mt, __shfl_xor(mt, 32));
            const float mn = fmaxf(m, mt), ms = mn == -INFINITY ? 0.f : mn, al = exp2_hw(m - ms), base = ms - one_lift<T>();
            m = mn;
            l *= al;
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] *= al;
#pragma unroll
            for (int kt = 0; kt < KT / 16; ++kt)
#pragma unroll
                for (int c = 0; c < 4; ++c) { sc[kt][c] = exp2_hw(sc[kt][c] - base); l += sc[kt][c]; }
            if constexpr (sizeof(T) == 2) {
                TwoParts<T> w;
#pragma unroll
                for (int c = 0; c < 8; ++c) w.set(c, sc[c >> 2][c & 3]);
#pragma unroll
                for (int i = 0; i < DT; ++i) {
                    const int r = 4 * g + (l15 >> 2), c = 2 * i + ((l15 >> 1) & 1), o = (l15 & 1) * 8;
                    s16x4 v[2] = {read_tr(vt_lds + TL::template voff<16>(r, c) + o), read_tr(vt_lds + TL::template voff<16>(r + 16, c) + o)};
                    auto vf = __builtin_bit_cast(typename Vec<T, 8>::type, v);
                    acc[i] = mma16(vf, w.upper, acc[i]);
                    if (odd) vf = finite_only(vf);
                    acc[i] = mma16(vf, w.rest, acc[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < DT; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float v = *(const float*)(vt_lds + TL::template voff<16>(4 * g + c, 4 * i + (l15 >> 2)) + (l15 & 3) * 4);
                        acc[i] = mma16(v, sc[0][c], acc[i]);
                    }
            }
        }
        // ---- the waves' parts joined: maxima and sums first, then each wave adds its scaled part
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (__any(lost)) l = NAN;
        __syncthreads();                                        // the tiles are free
        if (g == 0) { red_m[wave][l15] = m; red_l[wave][l15] = l; }
        float* sum = (float*)lds;                               // [16 rows][DP + 4]
        constexpr int SP = DP + 4;
        __syncthreads();
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, red_m[w][l15]);
        const float MS = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < NW; ++w) L += red_l[w][l15] * exp2_hw(red_m[w][l15] - MS);
        const float mine = exp2_hw(m - MS);
        for (int w = 0; w < NW; ++w) {
            if (wave == w)
#pragma unroll
                for (int i = 0; i < DT; ++i) {
                    f32x4* d = (f32x4*)(sum + l15 * SP + i * 16 + g * 4);
                    *d = w ? *d + acc[i] * mine : acc[i] * mine;
                }
            __syncthreads();
        }
        const bool whole = ua == 0 && ub == n_units;
        if (tid < 16) { red_m[0][tid] = M; red_l[0][tid] = L; }     // (each lane of the first 16 holds its own row's)
        __syncthreads();
        if (whole) {
            for (int i = tid; i < rows * Dh; i += 64 * NW) {
                const int r = i / Dh, d = i - r * Dh;
                ((T*)a.out)[((int64_t)s * p.Hq + h0 + r) * Dh + d] = (T)(sum[r * SP + d] / red_l[0][r]);
            }
        } else {
            float* o = a.part + ((int64_t)blockIdx.x * 2 + (ua == 0)) * piece_floats(DP);       // slot 0: began in an earlier share
            for (int i = tid; i < rows * DP; i += 64 * NW) o[i] = sum[(i / DP) * SP + i % DP];
            if (tid < rows) { o[ONE_ROWS * DP + tid] = red_m[0][tid]; o[ONE_ROWS * (DP + 1) + tid] = red_l[0][tid]; }
        }
        __syncthreads();
        u0 = seg0 + ub;
    }
}

// Adds the pieces of the segments that no block of attend_one had whole, in the order of the keys.  One block per segment and
// query head; the pieces' factors first, so that their rows are requested side by side.
template <typename T, int DP>
__global__ __launch_bounds__(DP) void attend_join(AttendArgs a, int keys) {
    __shared__ float factor[ONE_GRID];
    const PagedArgs& p = a.p;
    const int group = p.Hq / p.Hkv, rts = (group + 15) / 16, segs = p.Hkv * rts, lane = threadIdx.x & 63;
    const int s = blockIdx.x / segs, seg = blockIdx.x % segs, d = threadIdx.x, r = blockIdx.y;
    const int kvh = seg / rts, h0 = kvh * group + (seg - kvh * rts) * 16;
    if (r >= kvh * group + group - h0) return;
    const int n = Units::of_stream(p, s, keys);
    if (!n) return;
    Units U;
    U.sum(p, keys, segs);
    int64_t before = 0;
    for (int b = 0; b < s; b += 64) before += b + lane < s ? Units::of_stream(p, b + lane, keys) : 0;
    for (int o = 32; o; o >>= 1) before += __shfl_xor(before, o);
    const int64_t first = before * segs + (int64_t)seg * n;
    const int b0 = (int)(first / U.per), b1 = (int)((first + n - 1) / U.per);
    if (b0 == b1) return;
    auto piece_of = [&](int b) { return a.part + ((int64_t)b * 2 + (b == b0)) * piece_floats(DP); };
    float M = -INFINITY, L = 0.f;
    for (int b = b0 + lane; b <= b1; b += 64) M = fmaxf(M, piece_of(b)[ONE_ROWS * DP + r]);
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    const float MS = M == -INFINITY ? 0.f : M;
    for (int b = b0 + lane; b <= b1; b += 64) {
        const float* o = piece_of(b);
        const float f = exp2_hw(o[ONE_ROWS * DP + r] - MS);
        if (d < 64) factor[b - b0] = f;
        L += o[ONE_ROWS * (DP + 1) + r] * f;
    }
    for (int o = 32; o; o >>= 1) L += __shfl_xor(L, o);
    __syncthreads();
    float acc = 0.f;
#pragma unroll 8
    for (int b = b0; b <= b1; ++b) acc = fmaf(piece_of(b)[r * DP + d], factor[b - b0], acc);
    if (d < p.Dh) ((T*)a.out)[((int64_t)s * p.Hq + h0 + r) * p.Dh + d] = (T)(acc / L);
}

// ---- many rows per stream -------------------------------------------------------------------------------------------------
// A block's four waves have 32 rows each and share every tile of keys and values in LDS: two buffers, one barrier per tile, the
// next tile requested at the start of a tile and stored at its end.  Inside a wave the exponentials of 16 keys run under the
// matrix instructions of the 16 before them.  The blocks of a stream walk the keys side by side, so that L2 serves 93 % of what
// they read; equal shares of all the work, cut anywhere, would lose that (51 %) and 25 % of the speed.
// Bound by the order of work inside a wave: a tile of 64 keys x 128 dims takes the two waves of a SIMD about 5600 cycles, of which they
// keep its matrix pipe busy for 2048 (36 %) and its vector pipe for 44 %.  A wave issues for 40 % of its time, waits for its turn to issue
// for 32 % and for data and the barrier for 28 %: its scores, their maximum and the first weights stand in a line in front of the
// products with the values, and one other wave is too little to run under them.  5 streams of 100 to 8160 tokens, 16 heads on 4, bf16:
// 408 us, 800 TF (a large matrix product reaches 1224 TF); 16 streams of 512 tokens behind 4080, 8 heads on 2 x 64, fp32: 640 us,
// 114 TF (154): 96 % of the matrix rate inside the tiles, the rest goes into the start and end of blocks.
// 16-bit weights are rounded to the tensors' type for the product with the values: the result is off by 2.1e-3 of its size where one
// rounding to bf16 is 1.7e-3 (fp16: 2.5e-4, 2.1e-4).  In two parts, as attend_one has them, the 5 streams take 540 us.
// Two row sets per wave, or three waves per SIMD, spill; tiles of 32 keys, eight-wave blocks and staggered halves are slower.
template <typename T> constexpr int chunk_kt() { return sizeof(T) == 2 ? 64 : 32; }       // keys per tile
constexpr float LAZY = 8.f;         // the running maximum may lag by 2^8 before the sums are rescaled (weights up to 256: no loss)

// the larger of a lane's value and that of the lane 32 away
__device__ __forceinline__ float max_of_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float sum2(f16 a, f16 b, float x, float y, float l) { return l + x + y; }
__device__ __forceinline__ float sum2(bfl a, bfl b, float, float, float l) {
    typedef Vec<bfl, 2>::type B2;
    return __builtin_amdgcn_fdot2_f32_bf16(B2{a, b}, B2{(bfl)1.f, (bfl)1.f}, l, false);   // two rounded weights in one instruction
}

constexpr int CHUNK_WAVES = 4, CHUNK_ROWS = 32 * CHUNK_WAVES, CHUNK_EXTRA = 512;
template <typename T> constexpr int chunk_start() { return sizeof(T) == 4 ? 256 : 384; }    // keys' worth of time that a block takes to start and end
template <typename T> constexpr int chunk_least() { return sizeof(T) == 4 ? 64 : 256; }     // keys of a part, at least
// floats of a piece: a row tile's sums as [DP / 4][rows][4], then its maxima and sums of weights
constexpr int64_t chunk_piece(int DP) { return CHUNK_ROWS * (DP + 2); }

__device__ __forceinline__ int of_lane(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
struct ChunkStream {
    int start, rows, tiles, ahead;              // first packed row, rows, row tiles; keys before them, in those that a row tile adds
    __device__ __forceinline__ ChunkStream(const PagedArgs& p, int s) : start(0), rows(0), tiles(0), ahead(0) {
        if (s >= p.S) return;
        const int lo = p.offsets[s], hi = p.offsets[s + 1], past = p.lengths[s], group = p.Hq / p.Hkv;
        start = min(max(lo, 0), p.M);
        rows = max(0, min(hi, p.M) - start);
        tiles = (int)(((int64_t)rows * group + CHUNK_ROWS - 1) / CHUNK_ROWS);
        ahead = (int)min((int64_t)1 << 29, min((int64_t)max(past, 0), (int64_t)p.width << p.page_shift) * group / CHUNK_ROWS);
    }
};
// The work of up to 32 streams: their row tiles by the keys they look at, the most first, and the long ones in parts.  A stream's
// tile t has ahead + t + 1 units of keys; one of more than `part` units is cut.  Run by a whole wave, a lane a stream; uniform
// results, which depend on the lengths alone and are exact in every kernel (whole numbers and halves below 2^53).
// 4 x 510 tokens behind 1117 to 4080, 8 heads on 2 x 64, fp32: 133 us, 154 with every row tile in the same number of parts.  12 streams
// of 200 to 900 tokens behind up to 6000, 16 heads on 4 x 64, bf16: 70 to 113 us, 123 to 134 uncut.  It takes about 50 instructions per
// stream, twice: 64 streams of 4 tokens behind 2000, 8 heads on 2 x 64, fp16, would take 66 us with it and take 41 without.  More streams
// than 32 are not cut, which costs them dear where one is long: 4 tokens each, one stream behind 60000 and the others behind 500, bf16,
// take 61 us with 32 streams and 1032 with 33.
constexpr int CHUNK_STREAMS = 32, CHUNK_LEVELS = 64, CHUNK_SLOTS = 512;
struct ChunkPlan {
    const ChunkStream& c;
    int S, part;
    int level, upto;                            // lane j: tiles that have a part j; parts 1 to j of all tiles
    // tiles of more than so many units (a lane's own number)
    __device__ __forceinline__ int above(int units) const {
        int n = 0;
        for (int s = 0; s < S; ++s) {
            const int t = of_lane(c.tiles, s);
            n += max(0, min(t, of_lane(c.ahead, s) + t - units));
        }
        return n;
    }
    // The length of a part, `least` at least: of 63 of them, a lane's each, from a slot's fair share to five, and no cut at all, the one
    // that ends first - by the longest part where every part finds a slot at once, by the work of a slot and half a part where not -
    // with `start` units for the beginning of each.  Shares this long give fewer than `extra` parts beyond the tiles' first ones.
    __device__ __forceinline__ ChunkPlan(const ChunkStream& c, int S, int Hkv, int extra, int least, int start) : c(c), S(S), part(1 << 30) {
        const int lane = threadIdx.x & 63;
        if (extra) {
            double all = 0, parts = 0;
            int most = 1;
            for (int s = 0; s < S; ++s) {
                const int t = of_lane(c.tiles, s), a = of_lane(c.ahead, s);
                all += (double)t * (a + 0.5 * (t + 1));
                if (t) most = max(most, a + t);
            }
            all *= Hkv;
            const double share = all / extra * (lane + 16) / 16;
            const int floor = max(least, (most + CHUNK_LEVELS - 1) / CHUNK_LEVELS);
            const unsigned mine = lane == 63 || share > most ? most : max(floor, (int)share + 1);
            const float inv = __builtin_amdgcn_rcpf((float)mine);
            for (int s = 0; s < S; ++s) {       // of a stream, about: the shortest tile's and the longest's (1e-4: a whole number stays one)
                const int t = of_lane(c.tiles, s), a = of_lane(c.ahead, s);
                const float longest = ceilf(__builtin_fmaf((float)(a + t), inv, -1e-4f)), shortest = ceilf(__builtin_fmaf((float)(a + 1), inv, -1e-4f));
                parts += 0.5 * t * (double)(longest + shortest);
            }
            parts *= Hkv;
            const double cost = parts <= CHUNK_SLOTS ? (double)mine + start : (all + parts * start) / CHUNK_SLOTS + 0.5 * mine;
            double best = cost;
            for (int o = 32; o; o >>= 1) best = fmin(best, __shfl_xor(best, o));
            part = of_lane((int)mine, 63 - __clzll(__ballot(cost == best)));
        }
        level = above((int)min((int64_t)lane * part, (int64_t)1 << 30));
        upto = lane ? level : 0;
        for (int o = 1; o < 64; o <<= 1) { const int v = __shfl_up(upto, o); if (lane >= o) upto += v; }
    }
    __device__ __forceinline__ int tiles() const { return of_lane(level, 0); }
    __device__ __forceinline__ int cut() const { return of_lane(level, 1); }          // tiles in parts: the first so many
    __device__ __forceinline__ int beyond() const { return of_lane(upto, 63); }       // parts beyond the tiles' first ones
    // part number and place of the tile of the b-th of them
    __device__ __forceinline__ int part_of(int b, int& at) const {
        const int j = __ffsll(__ballot(upto > b)) - 1;
        at = b - of_lane(upto - level, j);
        return j;
    }
    // the tile in place `at` < tiles(): its stream and number.  64 thresholds at a time
    __device__ __forceinline__ int find(int at, int& tile) const {
        const int lane = threadIdx.x & 63;
        int lo = 0, hi = 0;                     // more than `at` tiles have over lo units, none has over hi
        for (int s = 0; s < S; ++s) hi = max(hi, of_lane(c.ahead, s) + of_lane(c.tiles, s));
        while (lo + 1 < hi) {
            const int step = (hi - lo - 1) / 64 + 1, units = lo + lane * step;
            const int b = 63 - __clzll(__ballot((above(units) > at) & (units < hi)));
            lo += b * step;
            hi = min(hi, lo + step);
        }
        int r = at - __builtin_amdgcn_readfirstlane(above(lo + 1));
        unsigned long long of = __ballot(lane < S && c.ahead <= lo && lo < c.ahead + c.tiles);
        while (r-- > 0) of &= of - 1;
        const int s = __ffsll(of) - 1;
        tile = lo - of_lane(c.ahead, s);
        return s;
    }
    __device__ __forceinline__ int parts(int units) const { return (units + part - 1) / part; }
};

template <typename T, int DP>
__global__ __launch_bounds__(64 * CHUNK_WAVES, (int)sizeof(T) * DP > 256 ? 1 : 2) void attend_chunk(AttendArgs a) {
    constexpr int KT = chunk_kt<T>(), NK = KT / 32, R = CHUNK_ROWS, NT = 64 * CHUNK_WAVES, DT = DP / 32;
    typedef Tile<T, DP> TL;
    constexpr int LD = KT * TL::CPR / NT, TILE_BYTES = KT * TL::PITCH;
    typedef typename Vec<T, 8>::type V8;
    extern __shared__ __attribute__((aligned(16))) char lds[];              // K x 2, V x 2, flags
    unsigned long long* flag = (unsigned long long*)(lds + 4 * TILE_BYTES); // [4]: rows of a V tile that held something not finite
    int* badf = (int*)(flag + 4);                                           // [4]: groups of 16 keys without a page
    const PagedArgs& p = a.p;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l31 = lane & 31, hf = lane >> 5;
    const int group = p.Hq / p.Hkv, Dh = p.Dh;
    const int kvh = blockIdx.x % p.Hkv, tile_id = blockIdx.x / p.Hkv;
    // ---- rows of no stream are 0
    if (kvh == 0) {
        const int lo = min(max(p.offsets[0], 0), p.M), hi = min(max(p.offsets[p.S], 0), p.M), none = lo + p.M - hi;
        for (int r = tile_id; r < none; r += gridDim.x / p.Hkv) {
            T* o = (T*)a.out + (int64_t)(r < lo ? r : hi + r - lo) * p.Hq * Dh;
            for (int i = tid; i < p.Hq * Dh; i += NT) o[i] = (T)0.f;
        }
    }
    // ---- stream and rows of this block, and which part of their keys: first the parts beyond the first of long row tiles, then all
    // row tiles, the longest first
    int s = -1, row0 = 0, n_rows = 0, start = 0, n_parts = 1, my_part = 0, slot = 0;
    if (p.S <= CHUNK_STREAMS) {
        const ChunkStream c(p, lane);
        const ChunkPlan plan(c, p.S, p.Hkv, a.extra, chunk_least<T>() * group / R + 1, chunk_start<T>() * group / R);
        int at;
        if (tile_id < plan.beyond()) {
            my_part = plan.part_of(tile_id, at);
            slot = plan.cut() + tile_id;                // of the pieces: the first parts of the cut tiles, then the others
        } else {
            slot = at = tile_id - plan.beyond();
            if (at >= plan.tiles()) return;
        }
        int tile;
        s = plan.find(at, tile);
        start = of_lane(c.start, s); n_rows = of_lane(c.rows, s) * group; row0 = tile * R;
        n_parts = plan.parts(of_lane(c.ahead, s) + tile + 1);
    } else {                                                                // the streams end to end, a stream's last (longest) tile first
        int64_t before = 0;
        for (int b = 0; b < p.S && s < 0; b += 64) {
            const ChunkStream c(p, b + lane);
            int64_t inc = c.tiles;
            for (int o = 1; o < 64; o <<= 1) { const int64_t v = __shfl_up(inc, o); if (lane >= o) inc += v; }
            const unsigned long long hit = __ballot(before + inc > tile_id);
            if (hit) {
                const int l = __ffsll(hit) - 1;
                s = b + l;
                start = of_lane(c.start, l);
                n_rows = of_lane(c.rows, l) * group;
                row0 = (int)(before + __shfl(inc, l) - 1 - tile_id) * R;
            } else before += __shfl(inc, 63);
        }
    }
    s = __builtin_amdgcn_readfirstlane(s);
    if (s < 0) return;
    row0 = __builtin_amdgcn_readfirstlane(row0); n_rows = __builtin_amdgcn_readfirstlane(n_rows); start = __builtin_amdgcn_readfirstlane(start);
    const int past = p.lengths[s];
    auto at = [&](int token) { return max(-1, paged_position(past, token)); };
    const int r = row0 + wave * 32 + l31, rr = min(r, n_rows - 1), tok = rr / group, h = kvh * group + rr - tok * group;
    const int pos = at(tok);                                                // this lane's row sees keys up to here
    const int b_lo = at(row0 / group), b_hi = at((min(row0 + R, n_rows) - 1) / group);
    int t_lo = 0, t_hi = b_hi < 0 ? 0 : (int)((paged_keys(p.width, p.page_shift, b_hi) - 1) / KT) + 1;
    if (n_parts > 1) {
        const int per = (t_hi + n_parts - 1) / n_parts;
        t_lo = min(t_hi, my_part * per); t_hi = min(t_hi, t_lo + per);
    }
    // ---- Q fragments
    u32x4 qf[TL::CPR / 2];
    const T* q = (const T*)a.q + (int64_t)(start + tok) * a.q_sm + h * a.q_sh;
#pragma unroll
    for (int i = 0; i < TL::CPR / 2; ++i) qf[i] = piece(q + (2 * i + hf) * TL::PER, (2 * i + hf) * TL::PER < Dh);
    f32x16 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int c = 0; c < 16; ++c) acc[i][c] = 0.f;
    float m = -INFINITY, l = 0.f;
    // ---- staging.  The 64 pieces that a wave requests at once lie in one group of 16 keys, hence in one page: their place is
    // scalar arithmetic, plus an offset of the lane's own that never changes.  Page numbers are looked up a tile before they are
    // used, by vector loads: a scalar load would be waited for together with the LDS reads
    u32x4 kr[LD], vr[LD];
    int entry[LD];                                                          // what the table holds for the next tile
    int grp[LD];                                                            // first key of the group
    unsigned k_off[LD], v_off[LD];
    const unsigned row_bytes = Dh * (unsigned)sizeof(T), page_mask = (1u << p.page_shift) - 1, table_keys = (unsigned)p.width << p.page_shift;
    const unsigned page_bytes = (p.Hkv << p.page_shift) * row_bytes;
    const char *k_pool = (const char*)a.k_pages + ((int64_t)kvh << p.page_shift) * row_bytes, *v_pool = (const char*)a.v_pages + ((int64_t)kvh << p.page_shift) * row_bytes;
#pragma unroll
    for (int j = 0; j < LD; ++j) {
        const int i = j * NT + tid, rw = i / TL::CPR, kc = TL::kswz(rw, i % TL::CPR) * TL::PER, vc = TL::template vswz<32>(rw, i % TL::CPR) * TL::PER;
        grp[j] = __builtin_amdgcn_readfirstlane(rw & ~15);
        k_off[j] = (rw & 15) * row_bytes + (kc < Dh ? kc : 0) * (unsigned)sizeof(T);
        v_off[j] = (rw & 15) * row_bytes + (vc < Dh ? vc : 0) * (unsigned)sizeof(T);
    }
    int lost = 0;                                                           // groups of the tile requested last that have no page
    const int* table = p.table + (int64_t)s * p.width;
    auto look = [&](int t) {
#pragma unroll
        for (int j = 0; j < LD; ++j) entry[j] = table[min(((unsigned)t * KT + grp[j] + (lane & 15)) >> p.page_shift, (unsigned)p.width - 1)];
    };
    // bytes into a pool of the group of keys from `key` on; one without a page reads page 0 (and is flagged)
    auto place = [&](unsigned key, int page, bool& here) -> int64_t {
        here = (unsigned)page < (unsigned)p.pages && key < table_keys;
        return (int64_t)((uint64_t)(unsigned)(here ? page : 0) * page_bytes) + (key & page_mask) * row_bytes;
    };
    // tile t; then the page numbers of tile t + 1.  Past the last tile too: in bounds, never used, and no branch around
    // loads in flight.  Keys behind the last one that a row sees are whatever their page holds (in bounds: a page ends behind
    // its last slot): their scores are masked, and store_v lets nothing through but numbers
    auto load = [&](int t) {
        lost = 0;
#pragma unroll
        for (int j = 0; j < LD; ++j) {
            bool here;
            const unsigned key = (unsigned)t * KT + grp[j];
            const int64_t where = place(key, __builtin_amdgcn_readfirstlane(entry[j]), here);
            lost |= (!here && key <= (unsigned)b_hi) << (grp[j] >> 4);
            kr[j] = *(const u32x4*)(k_pool + where + k_off[j]);
            vr[j] = *(const u32x4*)(v_pool + where + v_off[j]);
        }
        look(t + 1);
    };
    auto store_k = [&](int t) {
        if (Dh < DP)                                                        // dims past the head: zeros, as in Q
#pragma unroll
            for (int j = 0; j < LD; ++j) {
                const int i = j * NT + tid;
                if (TL::kswz(i / TL::CPR, i % TL::CPR) * TL::PER >= Dh) kr[j] = u32x4{0, 0, 0, 0};
            }
        char* to = lds + ((t - t_lo) & 1) * TILE_BYTES + tid * 16;
#pragma unroll
        for (int j = 0; j < LD; ++j) *(u32x4*)(to + j * NT * 16) = kr[j];
        if (lost && lane == 0) atomicOr(badf + ((t - t_lo) & 3), lost);
    };
    auto store_v = [&](int t) {
        if (b_lo - t * KT < KT - 1) {
            // not every row of the block sees the whole tile: a value that is not finite would reach those that do not see it
            // (0 x NaN).  It is stored as 0, and its key remembered
#pragma unroll
            for (int j = 0; j < LD; ++j) {
                bool odd = false;
#pragma unroll
                for (int k = 0; k < TL::PER; ++k) {
                    if constexpr (sizeof(T) == 4) {
                        f32x4 v = as<f32x4>(vr[j]);
                        if (!__builtin_isfinite(v[k])) { odd = true; v[k] = 0.f; vr[j] = __builtin_bit_cast(u32x4, v); }
                    } else {
                        V8 v = as<V8>(vr[j]);
                        if (!__builtin_isfinite((float)v[k])) { odd = true; v[k] = (T)0.f; vr[j] = __builtin_bit_cast(u32x4, v); }
                    }
                }
                if (odd) atomicOr(flag + ((t - t_lo) & 3), 1ull << ((j * NT + tid) / TL::CPR));
            }
        }
        char* to = lds + (2 + ((t - t_lo) & 1)) * TILE_BYTES + tid * 16;
#pragma unroll
        for (int j = 0; j < LD; ++j) *(u32x4*)(to + j * NT * 16) = vr[j];
    };
    auto tile = [&](int t, auto plain) __attribute__((always_inline)) {
        constexpr bool PLAIN = decltype(plain)::value;                      // every row of the block sees the whole tile, every key has a page
        const char *k_lds = lds + ((t - t_lo) & 1) * TILE_BYTES, *v_lds = k_lds + 2 * TILE_BYTES;
        load(t + 1);
        if (tid == 0) { flag[(t - t_lo + 2) & 3] = 0; badf[(t - t_lo + 2) & 3] = 0; }       // last read two barriers ago, next set behind the next
        // ---- scores: lane = (row l31, keys 8 b + 4 hf + 0..3 of each 32)
        f32x16 sc[NK];
#pragma unroll
        for (int kt = 0; kt < NK; ++kt)
#pragma unroll
            for (int c = 0; c < 16; ++c) sc[kt][c] = 0.f;
#pragma unroll
        for (int i = 0; i < TL::CPR / 2; ++i)
#pragma unroll
            for (int kt = 0; kt < NK; ++kt) {
                const u32x4 kf = *(const u32x4*)(k_lds + TL::koff(kt * 32 + l31, 2 * i + hf));
                if constexpr (sizeof(T) == 2) sc[kt] = mma32(as<V8>(kf), as<V8>(qf[i]), sc[kt]);
                else
#pragma unroll
                    for (int c = 0; c < 4; ++c) sc[kt] = mma32(as<f32x4>(kf)[c], as<f32x4>(qf[i])[c], sc[kt]);
            }
        if (!PLAIN) {
            const int bad = __builtin_amdgcn_readfirstlane(badf[(t - t_lo) & 3]);
            if (bad) {                                                      // scores of keys without a page: not a number
#pragma unroll
                for (int kt = 0; kt < NK; ++kt)
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        if (bad >> (kt * 2 + (c >> 3)) & 1) sc[kt][c] = NAN;
            }
            const int left = pos - t * KT - 4 * hf;                         // keys of the tile the row sees, from this lane's first on: 0 .. left
#pragma unroll
            for (int kt = 0; kt < NK; ++kt)
#pragma unroll
                for (int c = 0; c < 16; ++c) sc[kt][c] = left >= kt * 32 + 8 * (c >> 2) + (c & 3) ? sc[kt][c] : -INFINITY;
        }
        float mt = sc[0][0];
#pragma unroll
        for (int kt = 0; kt < NK; ++kt)
#pragma unroll
            for (int c = 0; c < 16; ++c) mt = fmaxf(mt, sc[kt][c]);
        mt = max_of_halves(mt) * a.scale_log2e;
        if (__any(mt > m + LAZY)) {
            const float mn = fmaxf(m, mt), al = exp2_hw(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= al;
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int c = 0; c < 16; ++c) acc[i][c] *= al;
        }
        const float ms = m == -INFINITY ? 0.f : m;
        if (!PLAIN) {
            // values that are not finite, of a tile that not every row sees whole: whatever its weight, such a one decides the sum
            const unsigned long long keys = flag[(t - t_lo) & 3];
            if (keys) {
#pragma nounroll
                for (int k = 0; k < KT; ++k) {
                    if (!(keys >> k & 1) || pos - t * KT < k) continue;
                    bool here;
                    const unsigned key = (unsigned)t * KT + k;
                    const T* v = (const T*)(v_pool + place(key, table[min(key >> p.page_shift, (unsigned)p.width - 1)], here)) + 4 * hf;
                    if (!here) continue;
#pragma unroll
                    for (int i = 0; i < DT; ++i)
#pragma unroll
                        for (int c = 0; c < 16; c += 4) {
                            typedef typename Vec<T, 4>::type V4;
                            const V4 x = i * 32 + 2 * c + 4 * hf < Dh ? *(const V4*)(v + i * 32 + 2 * c) : V4{};
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[i][c + e] += __builtin_isfinite((float)x[e]) ? 0.f : (float)x[e];
                        }
                }
            }
        }
        // ---- weights of 16 keys, and their values
#pragma unroll
        for (int k16 = 0; k16 < KT / 16; ++k16) {
            float w[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) w[c] = exp2_hw(fmaf(sc[k16 >> 1][(k16 & 1) * 8 + c], a.scale_log2e, -ms));
            if constexpr (sizeof(T) == 2) {
                V8 pf;                                                      // (rounded)
#pragma unroll
                for (int c = 0; c < 8; ++c) pf[c] = (T)w[c];
#pragma unroll
                for (int c = 0; c < 8; c += 2) l = sum2(pf[c], pf[c + 1], w[c], w[c + 1], l);
#pragma unroll
                for (int i = 0; i < DT; ++i) {
                    const int rw = k16 * 16 + 4 * hf + ((lane & 15) >> 2), c = 4 * i + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1), o = (lane & 1) * 8;
                    s16x4 v[2] = {read_tr(v_lds + TL::template voff<32>(rw, c) + o), read_tr(v_lds + TL::template voff<32>(rw + 8, c) + o)};
                    acc[i] = mma32(__builtin_bit_cast(V8, v), pf, acc[i]);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) l += w[c];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int rw = k16 * 16 + 8 * (c >> 2) + 4 * hf + (c & 3);
#pragma unroll
                    for (int i = 0; i < DT; ++i)
                        acc[i] = mma32(*(const float*)(v_lds + TL::template voff<32>(rw, 8 * i + (l31 >> 2)) + (l31 & 3) * 4), w[c], acc[i]);
                }
            }
        }
        store_k(t + 1);
        store_v(t + 1);
        __syncthreads();
    };
    if (tid < 4) { flag[tid] = 0; badf[tid] = 0; }
    __syncthreads();
    int t = t_lo;
    if (t_lo < t_hi) {
        look(t_lo);
        load(t_lo);
        store_k(t_lo);
        store_v(t_lo);
    }
    __syncthreads();
    // first the tiles that every row of the block sees whole, then the rest (and what follows a missing page)
    for (const int t_plain = min(t_hi, (int)(((unsigned)b_lo + 1) / KT)); t < t_plain; ++t) {
        if (__builtin_amdgcn_readfirstlane(badf[(t - t_lo) & 3])) break;
        tile(t, std::true_type{});
    }
    for (; t < t_hi; ++t) tile(t, std::false_type{});
    l += __shfl_xor(l, 32);
    if (n_parts > 1) {
        float* o = a.part + ((int64_t)slot * p.Hkv + kvh) * chunk_piece(DP);
        const int row = wave * 32 + l31;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int c4 = 0; c4 < 4; ++c4)
                *(f32x4*)(o + ((i * 8 + 2 * c4 + hf) * R + row) * 4) = f32x4{acc[i][4 * c4], acc[i][4 * c4 + 1], acc[i][4 * c4 + 2], acc[i][4 * c4 + 3]};
        if (hf == 0) { o[DP * R + row] = m; o[(DP + 1) * R + row] = l; }
        return;
    }
    if (r >= n_rows) return;
    const int64_t orow = (int64_t)(start + tok) * p.Hq + h;
    const float inv = 1.f / l;
    T* o = (T*)a.out + orow * Dh;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
            const int d = i * 32 + 8 * c4 + 4 * hf;
            typename Vec<T, 4>::type v;
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = (T)(pos < 0 ? 0.f : acc[i][4 * c4 + c] * inv);
            if (d < Dh) *(typename Vec<T, 4>::type*)(o + d) = v;
        }
}

// Adds the parts of the row tiles that were cut, in the order of the keys.  A block per place and 8 Q dims, a thread
// per row and 4 Q: where there are few row tiles, finer (2 tiles in 31 parts: 16 blocks of 8 batches of loads otherwise).
template <typename T, int DP, int Q>
__global__ __launch_bounds__(2 * CHUNK_ROWS) void attend_chunk_join(AttendArgs a) {
    constexpr int R = CHUNK_ROWS;
    const PagedArgs& p = a.p;
    const int group = p.Hq / p.Hkv, lane = threadIdx.x & 63, kvh = blockIdx.x % p.Hkv, at = blockIdx.x / p.Hkv;
    const ChunkStream c(p, lane);
    const ChunkPlan plan(c, p.S, p.Hkv, a.extra, chunk_least<T>() * group / R + 1, chunk_start<T>() * group / R);
    if (at >= plan.cut()) return;
    int tile;
    const int s = plan.find(at, tile), start = of_lane(c.start, s), n_rows = of_lane(c.rows, s) * group, parts = plan.parts(of_lane(c.ahead, s) + tile + 1);
    __shared__ int place[CHUNK_LEVELS];
    if (threadIdx.x < 64) place[lane] = lane ? plan.cut() + plan.upto - plan.level + at : at;
    __syncthreads();
    const int row = threadIdx.x % R, d4 = (blockIdx.y * 2 + threadIdx.x / R) * Q, r = tile * R + row;
    if (r >= n_rows || d4 * 4 >= p.Dh) return;
    auto piece_of = [&](int j) { return a.part + ((int64_t)place[j] * p.Hkv + kvh) * chunk_piece(DP); };
    float M = -INFINITY, L = 0.f;
#pragma unroll 4
    for (int j = 0; j < parts; ++j) M = fmaxf(M, piece_of(j)[DP * R + row]);
    const float MS = M == -INFINITY ? 0.f : M;
    f32x4 acc[Q] = {};
#pragma unroll 8 / Q
    for (int j = 0; j < parts; ++j) {
        const float* o = piece_of(j);
        const float f = exp2_hw(o[DP * R + row] - MS);
        L += o[(DP + 1) * R + row] * f;
#pragma unroll
        for (int k = 0; k < Q; ++k) acc[k] += *(const f32x4*)(o + ((d4 + k) * R + row) * 4) * f;
    }
    const int tok = r / group, pos = paged_position(p.lengths[s], tok);
    T* out = (T*)a.out + ((int64_t)(start + tok) * p.Hq + kvh * group + r - tok * group) * p.Dh + d4 * 4;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        typename Vec<T, 4>::type v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(pos < 0 ? 0.f : acc[k][e] / L);
        if ((d4 + k) * 4 < p.Dh) *(typename Vec<T, 4>::type*)(out + k * 4) = v;
    }
}

int padded_dim(int Dh) { return Dh <= 64 ? 64 : Dh <= 128 ? 128 : 256; }

int64_t chunk_tiles(const PagedArgs& p) { return (int64_t)p.M * (p.Hq / p.Hkv) / CHUNK_ROWS + p.S; }
// Parts beyond the first that all row tiles together may be cut into, by the table's width (the lengths are on the device).  A part
// costs a row (Dh + 2) floats written and read: as much as 250 keys' 16-bit products, little next to fp32 ones (a tile of 32 keys x
// 128 dims takes 4 us).  So parts have 256 or 64 keys at least (64 tokens behind 2000, 8 heads on 2 x 128, bf16: 20 us, 25 in parts of
// 512), and a table of fewer than six is not cut at all (2 streams of 512 tokens, 32 heads on 8 x 64: 16 us, 27 in two parts).
template <typename T> int chunk_extra(const PagedArgs& p) {
    const int64_t keys = (int64_t)p.width << p.page_shift;
    return p.S > CHUNK_STREAMS || keys < 6 * chunk_least<T>() ? 0 : CHUNK_EXTRA;
}
// A cache that cannot hold more than this is not worth a second launch: 8 streams of 100 or 500 tokens, 8 heads on 2 x 64, take 8.9 us
// with a block per segment and 13 in shares, of 1000 tokens 12 both ways, of 4000 35 and 13.
bool one_whole(const PagedArgs& p) { return ((int64_t)p.width << p.page_shift) <= 512; }

template <typename T, int DP> void run_one(AttendArgs a, hipStream_t s) {
    const PagedArgs& p = a.p;
    const int64_t segs = (int64_t)p.S * p.Hkv * ((p.Hq / p.Hkv + 15) / 16);
    constexpr int keys = one_nw<DP>() * one_kt<T>();
    a.splits = !one_whole(p);
    attend_one<T, DP><<<a.splits ? ONE_GRID : (unsigned)segs, 64 * one_nw<DP>(), 0, s>>>(a);
    if (a.splits) attend_join<T, DP><<<dim3((unsigned)segs, (unsigned)(p.Hq / p.Hkv < ONE_ROWS ? p.Hq / p.Hkv : ONE_ROWS)), DP, 0, s>>>(a, keys);
}
template <typename T, int DP> void run_chunk(AttendArgs a, hipStream_t s) {
    constexpr int bytes = 4 * chunk_kt<T>() * DP * (int)sizeof(T) + 48;
    static std::atomic<uint64_t> set;                           // devices (a bit each) that grant the kernel more LDS than the default
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return;               // (the error stays for the caller's check)
    if (dev > 63 || !(set.load(std::memory_order_relaxed) >> dev & 1)) {
        if (hipFuncSetAttribute((const void*)attend_chunk<T, DP>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return;
        if (dev < 64) set.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    a.extra = chunk_extra<T>(a.p);
    const int more = (a.extra + a.p.Hkv - 1) / a.p.Hkv;
    attend_chunk<T, DP><<<(unsigned)((chunk_tiles(a.p) + more) * a.p.Hkv), 64 * CHUNK_WAVES, bytes, s>>>(a);
    if (!a.extra) return;
    const unsigned places = (unsigned)(std::min<int64_t>(more, chunk_tiles(a.p)) * a.p.Hkv);
    if (places < 128) attend_chunk_join<T, DP, 1><<<dim3(places, DP / 8), 2 * CHUNK_ROWS, 0, s>>>(a);
    else attend_chunk_join<T, DP, 4><<<dim3(places, DP / 32), 2 * CHUNK_ROWS, 0, s>>>(a);
}
template <typename T, int DP> void run(const AttendArgs& a, hipStream_t s) {
    if (!a.p.offsets) run_one<T, DP>(a, s); else run_chunk<T, DP>(a, s);
}
template <typename T> void run_dim(const AttendArgs& a, hipStream_t s) {
    switch (padded_dim(a.p.Dh)) {
        case 64: run<T, 64>(a, s); break;
        case 128: run<T, 128>(a, s); break;
        default: run<T, 256>(a, s);
    }
}

}  // namespace

int64_t attend_workspace(const AttendArgs& a, int elem) {
    const int DP = padded_dim(a.p.Dh);
    if (!a.p.offsets) return one_whole(a.p) ? 0 : (int64_t)ONE_GRID * 2 * piece_floats(DP) * (int64_t)sizeof(float);
    const int extra = elem == ELEM_F32 ? chunk_extra<float>(a.p) : chunk_extra<f16>(a.p), more = (extra + a.p.Hkv - 1) / a.p.Hkv;
    return extra ? (int64_t)2 * more * a.p.Hkv * chunk_piece(DP) * (int64_t)sizeof(float) : 0;
}
void launch_attend(AttendArgs a, int elem, hipStream_t s) {
    if (elem == ELEM_F32) run_dim<float>(a, s);
    else if (elem == ELEM_F16) run_dim<f16>(a, s);
    else run_dim<bfl>(a, s);
}
