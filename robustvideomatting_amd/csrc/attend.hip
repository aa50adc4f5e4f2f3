// Attention of new tokens over a paged key-value cache.
#include "temporal.hpp"

namespace {

// One wave per (row, query head), 64 keys at a time: a lane scores one key, then every lane sums its dims over the 64.
template <typename T>
__global__ __launch_bounds__(64) void attend_rows(AttendArgs a) {
    __shared__ float qs[256];
    __shared__ float ps[64];
    const int m = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const PagedArgs& p = a.p;
    const int Dh = p.Dh, kvh = h / (p.Hq / p.Hkv);
    int pos;
    const int s = __builtin_amdgcn_readfirstlane(paged_row(p, m, pos));
    T* out = (T*)a.out + ((int64_t)m * p.Hq + h) * Dh;
    if (s >= p.S || pos < 0) {
        for (int d = lane; d < Dh; d += 64) out[d] = (T)0.f;
        return;
    }
    for (int d = lane; d < Dh; d += 64) qs[d] = (float)((const T*)a.q)[m * a.q_sm + h * a.q_sh + d];
    __syncthreads();
    float mx = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int pmask = (1 << p.page_shift) - 1;
    for (int64_t j0 = 0; j0 <= pos; j0 += 64) {
        const int64_t j = j0 + lane;
        float sc = -INFINITY;
        int64_t base = -1;
        if (j <= pos) {
            const int pg = paged_page(p, s, (int)j);
            if (pg >= 0) {
                base = ((((int64_t)pg * p.Hkv + kvh) << p.page_shift) + (j & pmask)) * Dh;
                float d0 = 0.f;
                for (int d = 0; d < Dh; ++d) d0 += qs[d] * (float)((const T*)a.k_pages)[base + d];
                sc = d0 * a.scale_log2e;
            } else sc = NAN;
        }
        float tm = sc;
        for (int o = 32; o; o >>= 1) tm = fmaxf(tm, __shfl_xor(tm, o));
        const float mn = fmaxf(mx, tm), ms = mn == -INFINITY ? 0.f : mn;
        const float pr = exp2f(sc - ms), al = exp2f(mx - ms);
        float ts = pr;
        for (int o = 32; o; o >>= 1) ts += __shfl_xor(ts, o);
        l = l * al + ts;
        mx = mn;
        for (int k = 0; k < 4; ++k) acc[k] *= al;
        ps[lane] = pr;
        __syncthreads();
        for (int i = 0; i < 64 && j0 + i <= pos; ++i) {
            const int64_t b = ((int64_t)__shfl((int)(base >> 32), i) << 32) | (unsigned)__shfl((int)base, i);
            if (b < 0) continue;
            for (int k = 0; k < 4; ++k)
                if (lane + 64 * k < Dh) acc[k] += ps[i] * (float)((const T*)a.v_pages)[b + lane + 64 * k];
        }
        __syncthreads();
    }
    for (int k = 0; k < 4; ++k)
        if (lane + 64 * k < Dh) out[lane + 64 * k] = (T)(acc[k] / l);
}

}  // namespace

int64_t attend_workspace(const AttendArgs&, int) { return 0; }
void launch_attend(AttendArgs a, int elem, hipStream_t s) {
    const dim3 g(a.p.M, a.p.Hq);
    if (elem == ELEM_F32) attend_rows<float><<<g, 64, 0, s>>>(a);
    else if (elem == ELEM_F16) attend_rows<f16><<<g, 64, 0, s>>>(a);
    else attend_rows<bfl><<<g, 64, 0, s>>>(a);
}
