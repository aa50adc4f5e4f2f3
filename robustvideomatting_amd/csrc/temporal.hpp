// Temporal operators beside the recurrent decoder: argument blocks of the kernels in scan.hip, paged.hip and attend.hip
// (host checks and the C entries: temporal.cpp).  All of them are one recurrence over a stream in two forms - a chunk of
// steps, or one step - with the state (scan state, conv window, pages) owned by the caller.
#pragma once
#include "common.hpp"
#include "paged_index.hpp"

enum ElemType { ELEM_F32 = 0, ELEM_F16 = 1, ELEM_BF16 = 2 };
typedef __bf16 bfl;                                     // the compiler's bfloat16: conversions are one instruction on gfx950

template <typename T, int N> struct Vec { typedef T type __attribute__((ext_vector_type(N))); };

struct CausalConvArgs {
    const void *x, *weight, *bias, *state_in;           // [B,T,D] by strides, [W,D], [D] or null, [B,W-1,D] or null (zeros)
    void *y, *state_out;                                // [B,T,D], [B,W-1,D] dense
    int64_t x_sb, x_st;
    int B, T, D, W, silu, runs;
};
void launch_causal_conv(const CausalConvArgs& a, int elem, hipStream_t s);

struct ScanArgs {
    const void *x, *dt, *z, *Bm, *Cm;                   // z may be null
    const float *A, *D, *dt_bias, *state_in;            // [N,D]; the other three may be null
    void* y; float* state_out;                          // [B,T,D], [B,N,D]
    float *carry, *steps, *totals;                      // time split: [B][chunks][N][D] states, [B][chunks][D] sums of step sizes, of blocks
    int64_t x_sb, x_st, dt_sb, dt_st, z_sb, z_st, B_sb, B_st, C_sb, C_st;
    int B, T, nD, N, softplus, chunks, chunk_len, dtiles;
};
// how the time axis is split for this shape (1: not at all)
int scan_chunks(int B, int T, int D, int N);
int64_t scan_workspace_floats(int64_t B, int64_t chunks, int64_t D, int64_t N);
void launch_selective_scan(const ScanArgs& a, int elem, hipStream_t s);

// A stream's cache: position p lives in page table[s][p / page], slot p % page, of the pools [pages][Hkv][page][Dh]
struct PagedArgs {
    const int *table, *lengths, *offsets;               // [S][width], [S], [S+1] or null (row m is stream m's one token)
    int S, M, pages, page_shift, width, Hq, Hkv, Dh;
};
struct AppendArgs {
    PagedArgs p;
    const void *q, *k, *v; void *q_out, *k_pages, *v_pages; const float* freqs;     // q / q_out may be null
    int64_t q_sm, q_sh, k_sm, k_sh, v_sm, v_sh;
    int rot, interleaved;                               // rot: rotated dims (twice the number of freqs)
};
void launch_append_kv(const AppendArgs& a, int elem, hipStream_t s);

struct AttendArgs {
    PagedArgs p;
    const void *q, *k_pages, *v_pages; void* out;       // out [M][Hq][Dh]
    int64_t q_sm, q_sh;
    float scale_log2e;                                  // softmax runs in base 2
    float* part; int splits, extra;                     // workspace; single tokens in shares; parts beyond the first of row tiles
};
int64_t attend_workspace(const AttendArgs& a, int elem);
void launch_attend(AttendArgs a, int elem, hipStream_t s);

#ifdef __HIPCC__
// Stream and position of packed row m, found by the whole wave (offsets are read 64 at a time).  stream == S: the row
// belongs to nobody.  Whatever the offsets hold, stream stays in [0, S]; a row in front of its stream's start is nobody's too.
__device__ __forceinline__ int paged_row(const PagedArgs& p, int m, int& pos) {
    int s = m, i = 0;
    if (p.offsets) {
        const int lane = threadIdx.x & 63;
        s = 0;
        for (int b = 0; b < p.S; b += 64) {
            const bool past = b + lane < p.S && p.offsets[b + lane + 1] <= m;
            s += __popcll(__ballot(past));
        }
        if (s < p.S) i = m - p.offsets[s];
        if (i < 0) s = p.S;
    }
    pos = s < p.S ? paged_position(p.lengths[s], i) : -1;
    return s;
}
__device__ __forceinline__ int paged_page(const PagedArgs& p, int s, int pos) {
    return page_of(p.table, p.width, p.pages, p.page_shift, s, pos);
}
#endif
