// ibh_lora.hip -- low-rank adapters of many requests beside a shared
// projection: out[b] = base[b] + scale * B (A x[b]) with the adapter of row b.
#include "ibh_common.h"

namespace {
using namespace ibh;

__device__ unsigned int ibh_lora_err;

struct Lora {
    const uint16_t *a, *b;
    const float* scales;
    const int32_t* ranks;
    int n, R, N, M, kind;
    float* out;
    const float *base, *x;
    const int32_t* ids;
    int B;
    size_t os, bs, xs;
    float* t;                                            // [B][R]: scale * A x
};

__device__ __forceinline__ float widen(uint16_t h, int kind) {
    return kind == IBH_F16 ? f16_to_f32(h) : __builtin_bit_cast(float, (uint32_t)h << 16);
}
// The rank of adapter `id`; -1 where the table does not have it.
__device__ __forceinline__ int rank_of(const Lora& l, int id) {
    if (id >= l.n) return -1;
    const int r = l.ranks ? l.ranks[id] : l.R;
    return r > l.R ? -1 : r < 0 ? -1 : r;
}

__global__ __launch_bounds__(256) void lora_shrink_kernel(Lora l) {
    const int row = blockIdx.x;
    const int id = l.ids[row];
    if (id < 0) return;
    const int rank = rank_of(l, id);
    const float scale = rank > 0 && l.scales ? l.scales[id] : 1.f;
    for (int r = blockIdx.y * 4 + (threadIdx.x >> 6); r < rank; r += gridDim.y * 4) {
        const uint16_t* a = l.a + ((size_t)id * l.R + r) * l.N;
        const float* x = l.x + row * l.xs;
        float s = 0;
        for (int j = threadIdx.x & 63; j < l.N; j += 64) s = fmaf(widen(a[j], l.kind), x[j], s);
        s = wave_sum(s);
        if ((threadIdx.x & 63) == 0) l.t[(size_t)row * l.R + r] = s * scale;
    }
}

__global__ __launch_bounds__(256) void lora_expand_kernel(Lora l) {
    const int row = blockIdx.x;
    const int id = l.ids[row];
    const int rank = id < 0 ? 0 : rank_of(l, id);
    if (rank < 0 && threadIdx.x == 0 && blockIdx.y == 0) atomicOr(&ibh_lora_err, IBH_DEVERR_LORA);
    for (int m = blockIdx.y * 256 + threadIdx.x; m < l.M; m += gridDim.y * 256) {
        float s = 0;
        for (int r = 0; r < rank; r++)
            s = fmaf(widen(l.b[((size_t)id * l.M + m) * l.R + r], l.kind), l.t[(size_t)row * l.R + r], s);
        if (l.base) s += l.base[row * l.bs + m];
        l.out[row * l.os + m] = rank < 0 ? __builtin_nanf("") : s;
    }
}

bool adapters_ok(const ibh_lora_adapters* l, const char* who) {
    if (!l || !l->a || !l->b || l->n <= 0 || l->rank <= 0 || l->rank > IBH_LORA_MAX_RANK || l->N <= 0 || l->M <= 0 ||
        l->N > (1 << 20) || l->M > (1 << 20) || (l->kind != IBH_F16 && l->kind != IBH_BF16)) {
        if (!l) ibh_set_error("%s: no adapters given", who);
        else
            ibh_set_error("%s: invalid adapters (n=%d rank=%d N=%d M=%d kind=%d; rank up to %d, IBH_F16 or IBH_BF16)",
                          who, l->n, l->rank, l->N, l->M, l->kind, IBH_LORA_MAX_RANK);
        return false;
    }
    return true;
}

}  // namespace

void* ibh_workspace(size_t bytes);

int ibh_lora_errors(bool clear) {
    unsigned int v = 0;
    if (hipMemcpyFromSymbol(&v, HIP_SYMBOL(ibh_lora_err), sizeof(v)) != hipSuccess) return -1;
    if (clear && v) {
        const unsigned int z = 0;
        if (hipMemcpyToSymbol(HIP_SYMBOL(ibh_lora_err), &z, sizeof(z)) != hipSuccess) return -1;
    }
    return (int)v;
}

extern "C" size_t ibh_lora_workspace_bytes(const ibh_lora_adapters* l, int B) {
    if (!adapters_ok(l, "ibh_lora_workspace_bytes") || B <= 0) return 0;
    return (size_t)B * l->rank * 4;
}

extern "C" int ibh_lora(const ibh_lora_adapters* l, float* out, const float* base, const float* x, const int32_t* ids,
                        int B, int out_stride, int base_stride, int x_stride, void* ws, size_t ws_bytes, void* stream) {
    if (!adapters_ok(l, "ibh_lora")) return IBH_ERROR_PARAM;
    if (B == 0) return IBH_OK;
    if (!out || !x || !ids || B < 0 || (B > 1 && (out_stride < l->M || (base && base_stride < l->M) || x_stride < l->N))) {
        ibh_set_error("ibh_lora: invalid arguments (B=%d out_stride=%d base_stride=%d x_stride=%d)", B, out_stride,
                      base_stride, x_stride);
        return IBH_ERROR_PARAM;
    }
    const size_t rows = B, ob = ((rows - 1) * out_stride + l->M) * 4, bb = ((rows - 1) * base_stride + l->M) * 4;
    const size_t xb = ((rows - 1) * x_stride + l->N) * 4, n = l->n;
    if (ibh_overlap(out, ob, x, xb) || (!(out == base && (B == 1 || out_stride == base_stride)) && ibh_overlap(out, ob, base, bb)) ||
        ibh_overlap(out, ob, ids, rows * 4) || ibh_overlap(out, ob, l->a, n * l->rank * l->N * 2) ||
        ibh_overlap(out, ob, l->b, n * l->rank * l->M * 2) || ibh_overlap(out, ob, l->scales, n * 4) ||
        ibh_overlap(out, ob, l->ranks, n * 4)) {
        ibh_set_error("ibh_lora: out overlaps another operand");
        return IBH_ERROR_PARAM;
    }
    if (B >= (1 << 24)) {
        ibh_set_error("ibh_lora: %d rows are more than one launch takes", B);
        return IBH_ERROR_PARAM;
    }
    const size_t need = ibh_lora_workspace_bytes(l, B);
    float* t = (float*)(ws ? (ws_bytes >= need && !((uintptr_t)ws & 15) ? ws : nullptr) : ibh_workspace(need));
    if (!t) {
        ibh_set_error("ibh_lora: a workspace of %zu bytes on 16 bytes is needed", need);
        return IBH_ERROR_MEMORY;
    }
    const Lora a{(const uint16_t*)l->a, (const uint16_t*)l->b, l->scales, l->ranks, l->n, l->rank, l->N, l->M, l->kind,
                 out, base, x, ids, B, (size_t)out_stride, (size_t)base_stride, (size_t)x_stride, t};
    hipStream_t st = ibh_resolve_stream(stream);
    lora_shrink_kernel<<<dim3(B, B > 1024 ? 1 : (l->rank + 3) / 4), 256, 0, st>>>(a);
    IBH_CHECK_LAUNCH("ibh_lora");
    lora_expand_kernel<<<dim3(B, B > 1024 ? 1 : (l->M + 255) / 256), 256, 0, st>>>(a);
    IBH_CHECK_LAUNCH("ibh_lora");
    return IBH_OK;
}
