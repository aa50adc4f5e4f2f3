// Which steps of its inputs a wave of the selective scan reads.  Plain C++ on both sides, so that the bounds can be checked on the host.
#pragma once
#include <stdint.h>
#ifndef RVM_HD
#ifdef __HIPCC__
#define RVM_HD __host__ __device__ __forceinline__
#else
#define RVM_HD inline
#endif
#endif
// Steps requested ahead, half of them for many states: 4 spill (58 x 171 x 99, 64 states: 79 us, not 61)
constexpr int SCAN_BATCH = 4;
RVM_HD constexpr int scan_batch(int NP, int PACK) { return NP * PACK <= 16 ? SCAN_BATCH : SCAN_BATCH / 2; }
// values of B (and C, but where only the chunks' ends are wanted) per step and sequence, and how many of a batch a lane holds
RVM_HD constexpr int scan_values(int NP, bool ends) { return ends ? NP : 2 * NP; }
RVM_HD constexpr int scan_loads(int NP, int PACK, bool ends) { return (scan_batch(NP, PACK) * PACK * scan_values(NP, ends) + 63) / 64; }
// Step of the batch that place e of 64 x scan_loads is dealt.  A batch may have fewer values than places (4 steps of 8): the places
// behind its last value have values of its last step, so that a wave reads no step behind its batch
RVM_HD constexpr int scan_step_of(int e, int NP, int PACK, bool ends) {
    const int k = e / (scan_values(NP, ends) * PACK), last = scan_batch(NP, PACK) - 1;
    return k < last ? k : last;
}
// Steps of a chunk: whole batches of loads
RVM_HD int64_t scan_chunk_len(int64_t T, int64_t chunks) { return ((T + chunks - 1) / chunks + SCAN_BATCH - 1) / SCAN_BATCH * SCAN_BATCH; }
// First step of a chunk and the one behind its last (both T where it has none); T and the length are below 2^31, their sums are not
RVM_HD int scan_first_step(int T, int chunk_len, int chunk) {
    const int64_t t = (int64_t)chunk * chunk_len;
    return t < T ? (int)t : T;
}
RVM_HD int scan_end_step(int T, int chunk_len, int first) { return T - first > chunk_len ? first + chunk_len : T; }
