// C entries of the temporal operators (include/rvm_mi355x.h): argument checks, then one to three launches on the caller's
// stream and the calling thread's current device.
#include "temporal.hpp"
#include "../../include/rvm_mi355x.h"

#include <cmath>
#include <cstring>
#include <string>

int rvm_set_error(const std::string& m);                // engine.cpp: the thread's rvm_last_error

namespace {

int fail(const char* who, const char* what) { return rvm_set_error(std::string(who) + ": " + what); }
int launched(const char* who) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail(who, hipGetErrorString(e));
}
int elem_of(int dtype) {
    switch (dtype) {
        case RVM_DTYPE_F32: return ELEM_F32;
        case RVM_DTYPE_F16: case RVM_DTYPE_F16IO: return ELEM_F16;
        case RVM_DTYPE_BF16IO: return ELEM_BF16;
        default: return -1;
    }
}
constexpr int64_t INT_LIMIT = 0x7fffffff, THREAD_LIMIT = 0xffffffff;     // of a launch, in one direction
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int paged_check(const char* who, PagedArgs& p, const int32_t* table, const int32_t* lengths, const int32_t* offsets, int64_t M, int64_t S,
                int64_t Hq, int64_t Hkv, int64_t Dh, int64_t pages, int64_t page, int64_t width) {
    if (M < 0 || S < 0 || M > INT_LIMIT || S > INT_LIMIT) return fail(who, "bad number of rows or streams");
    if (!offsets && M != S) return fail(who, "without offsets every stream has one row");
    if (M && !S) return fail(who, "rows for no stream");
    if (Hkv < 1 || Hq < 1 || Hq > 65535 || Hq % Hkv) return fail(who, "the query heads must be a multiple of the key heads");
    if (Dh < 8 || Dh > 256 || Dh % 8) return fail(who, "head size must be a multiple of 8, at most 256");
    if (page < 16 || page > 1024 || (page & (page - 1))) return fail(who, "page size must be a power of two from 16 to 1024");
    if (pages < 1 || pages > INT_LIMIT || width < 1 || width > INT_LIMIT || width * page > INT_LIMIT + 1) return fail(who, "bad page pool or table");
    if (Hkv * page * Dh > INT_LIMIT / 4) return fail(who, "bad page pool or table: a page of all heads must stay below 2 GiB in fp32");
    // what the kernels launch for M rows of S streams: at most 256 threads a row, a tile of 128 rows, or a (stream, key head, 16 heads)
    if (M * 256 > THREAD_LIMIT || M * Hq > INT_LIMIT / 4 || S * Hkv * ((Hq / Hkv + 15) / 16) * 256 > THREAD_LIMIT / 2) return fail(who, "too large for one launch");
    if (M && (!table || !lengths)) return fail(who, "null table or lengths");
    memset(&p, 0, sizeof p);
    p.table = table; p.lengths = lengths; p.offsets = offsets;
    p.S = (int)S; p.M = (int)M; p.pages = (int)pages; p.width = (int)width; p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.Dh = (int)Dh;
    while ((1 << p.page_shift) < page) ++p.page_shift;
    return 0;
}

}  // namespace

extern "C" {

int rvm_causal_conv(int dtype, const rvm_conv_args* c, void* hip_stream) {
    const char* who = "rvm_causal_conv";
    const int elem = elem_of(dtype);
    if (!c) return fail(who, "null arguments");
    if (elem < 0) return fail(who, "bad dtype");
    if (c->B < 0 || c->T < 0 || c->D < 0 || c->B > INT_LIMIT || c->T > INT_LIMIT - 64 || c->D > INT_LIMIT) return fail(who, "bad shape");
    if (c->W < 2 || c->W > 4) return fail(who, "the filter has 2 to 4 taps");
    if (!c->B || !c->D) return 0;
    if (!c->weight || !c->state_out || (c->T && (!c->x || !c->y))) return fail(who, "null buffer");
    if (c->state_in == c->state_out) return fail(who, "state_out must not alias state_in");
    if ((double)c->B * (c->T < 8 ? c->T + 1 : c->T / 8 + 1) * c->D > 4e9) return fail(who, "too large for one launch");
    CausalConvArgs a; memset(&a, 0, sizeof a);
    a.x = c->x; a.weight = c->weight; a.bias = c->bias; a.state_in = c->state_in; a.y = c->y; a.state_out = c->state_out;
    a.x_sb = c->x_sb; a.x_st = c->x_st; a.B = (int)c->B; a.T = (int)c->T; a.D = (int)c->D; a.W = (int)c->W; a.silu = c->silu != 0;
    launch_causal_conv(a, elem, (hipStream_t)hip_stream);
    return launched(who);
}

int64_t rvm_selective_scan_workspace(int64_t B, int64_t T, int64_t D, int64_t N) {
    if (B < 0 || T < 0 || D < 0 || N < 1 || B > INT_LIMIT || T > INT_LIMIT || D > INT_LIMIT || N > 64) return -1;
    if (!B || !D) return 0;
    const int64_t chunks = scan_chunks((int)B, (int)T, (int)D, (int)N);
    return chunks > 1 ? scan_workspace_floats(B, chunks, D, N) * (int64_t)sizeof(float) : 0;
}

int rvm_selective_scan(int dtype, const rvm_scan_args* c, void* hip_stream) {
    const char* who = "rvm_selective_scan";
    const int elem = elem_of(dtype);
    if (!c) return fail(who, "null arguments");
    if (elem < 0) return fail(who, "bad dtype");
    if (c->nB < 0 || c->nT < 0 || c->nD < 0 || c->nB > INT_LIMIT || c->nT > INT_LIMIT - 64 || c->nD > INT_LIMIT) return fail(who, "bad shape");
    if (c->nN < 1 || c->nN > 64) return fail(who, "1 to 64 states per channel");
    if (!c->nB || !c->nD) return 0;
    if (!c->A || !c->state_out || (c->nT && (!c->x || !c->dt || !c->B || !c->C || !c->y))) return fail(who, "null buffer");
    // (a row's bytes are a lane's 32-bit offset)
    if (c->nB * ((c->nD + 63) / 64) > THREAD_LIMIT / 128 || c->nD * (elem == ELEM_F32 ? 4 : 2) > THREAD_LIMIT + 1) return fail(who, "too large for one launch");
    if (c->state_in == c->state_out) return fail(who, "state_out must not alias state_in");
    const int64_t need = rvm_selective_scan_workspace(c->nB, c->nT, c->nD, c->nN);
    if (need > 0 && (!c->workspace || c->workspace_bytes < need)) return fail(who, "workspace too small (rvm_selective_scan_workspace)");
    ScanArgs a; memset(&a, 0, sizeof a);
    a.x = c->x; a.dt = c->dt; a.z = c->z; a.Bm = c->B; a.Cm = c->C;
    a.A = c->A; a.D = c->D; a.dt_bias = c->dt_bias; a.state_in = c->state_in; a.y = c->y; a.state_out = c->state_out;
    a.x_sb = c->x_sb; a.x_st = c->x_st; a.dt_sb = c->dt_sb; a.dt_st = c->dt_st; a.z_sb = c->z_sb; a.z_st = c->z_st;
    a.B_sb = c->B_sb; a.B_st = c->B_st; a.C_sb = c->C_sb; a.C_st = c->C_st;
    a.B = (int)c->nB; a.T = (int)c->nT; a.nD = (int)c->nD; a.N = (int)c->nN; a.softplus = c->softplus != 0;
    a.chunks = scan_chunks(a.B, a.T, a.nD, a.N);
    a.carry = (float*)c->workspace;
    launch_selective_scan(a, elem, (hipStream_t)hip_stream);
    return launched(who);
}

int rvm_append_kv(int dtype, const rvm_append_args* c, void* hip_stream) {
    const char* who = "rvm_append_kv";
    const int elem = elem_of(dtype);
    if (!c) return fail(who, "null arguments");
    if (elem < 0) return fail(who, "bad dtype");
    AppendArgs a; memset(&a, 0, sizeof a);
    if (int rc = paged_check(who, a.p, c->table, c->lengths, c->offsets, c->M, c->S, c->Hq, c->Hkv, c->Dh, c->pages, c->page, c->width)) return rc;
    if (c->rot < 0 || c->rot > c->Dh || c->rot % 16) return fail(who, "rotated dims must be a multiple of 16, at most the head size");
    if (!c->M) return 0;
    if (!c->k || !c->v || !c->k_pages || !c->v_pages || (c->rot && !c->freqs) || (c->q != nullptr) != (c->q_out != nullptr)) return fail(who, "null buffer");
    const int64_t v = elem == ELEM_F32 ? 4 : 8;
    if (!aligned16(c->q) || !aligned16(c->k) || !aligned16(c->v) || !aligned16(c->q_out) || !aligned16(c->k_pages) || !aligned16(c->v_pages) ||
        c->k_sm % v || c->k_sh % v || c->v_sm % v || c->v_sh % v || (c->q && (c->q_sm % v || c->q_sh % v)))
        return fail(who, "rows and heads must start on 16-byte boundaries");
    a.q = c->q; a.k = c->k; a.v = c->v; a.q_out = c->q_out; a.k_pages = c->k_pages; a.v_pages = c->v_pages; a.freqs = c->freqs;
    a.q_sm = c->q_sm; a.q_sh = c->q_sh; a.k_sm = c->k_sm; a.k_sh = c->k_sh; a.v_sm = c->v_sm; a.v_sh = c->v_sh;
    a.rot = (int)c->rot; a.interleaved = c->interleaved != 0;
    launch_append_kv(a, elem, (hipStream_t)hip_stream);
    return launched(who);
}

static int attend_prepare(const char* who, int dtype, const rvm_attend_args* c, AttendArgs& a, int& elem) {
    elem = elem_of(dtype);
    if (!c) return fail(who, "null arguments");
    if (elem < 0) return fail(who, "bad dtype");
    memset(&a, 0, sizeof a);
    if (int rc = paged_check(who, a.p, c->table, c->lengths, c->offsets, c->M, c->S, c->Hq, c->Hkv, c->Dh, c->pages, c->page, c->width)) return rc;
    const float scale = (float)(c->scale * 1.4426950408889634);
    if (!(scale > 0.f) || !std::isfinite(scale)) return fail(who, "scale must be positive and finite in fp32");
    a.q = c->q; a.k_pages = c->k_pages; a.v_pages = c->v_pages; a.out = c->out; a.q_sm = c->q_sm; a.q_sh = c->q_sh;
    a.scale_log2e = scale;
    return 0;
}

int64_t rvm_attend_workspace(int dtype, const rvm_attend_args* c) {
    AttendArgs a; int elem;
    if (attend_prepare("rvm_attend_workspace", dtype, c, a, elem)) return -1;
    return a.p.M ? attend_workspace(a, elem) : 0;
}

int rvm_attend(int dtype, const rvm_attend_args* c, void* hip_stream) {
    const char* who = "rvm_attend";
    AttendArgs a; int elem;
    if (int rc = attend_prepare(who, dtype, c, a, elem)) return rc;
    if (!c->M) return 0;
    if (!c->q || !c->k_pages || !c->v_pages || !c->out) return fail(who, "null buffer");
    const int64_t v = elem == ELEM_F32 ? 4 : 8;
    if (!aligned16(c->q) || !aligned16(c->k_pages) || !aligned16(c->v_pages) || !aligned16(c->out) || c->q_sm % v || c->q_sh % v)
        return fail(who, "rows and heads must start on 16-byte boundaries");
    const int64_t need = attend_workspace(a, elem);
    if (need > 0 && (!c->workspace || c->workspace_bytes < need || !aligned16(c->workspace))) return fail(who, "workspace too small (rvm_attend_workspace)");
    a.part = (float*)c->workspace;
    launch_attend(a, elem, (hipStream_t)hip_stream);
    return launched(who);
}

}  // extern "C"
