// ibh_norm.hip -- the residual's addition, the RMS norm and its 8-bit codes
// for a batch of rows in one pass.
//
// Memory bounds it: x and delta come once, h and y or the codes go once.  4099
// rows of 4096 with h and y, 269 MB, take 43 us (6.2 TB/s; a plain copy of a
// gigabyte runs at 5.2), with codes 37, with y and codes 49 us; 512 rows with codes
// 8.0 us; one row 3 us, of which a launch is 2 (kernels, traced one by one; a row
// of calls with h and y takes 47 us each).  The sums in 64 bits cost nothing beside
// that.
#include "ibh_common.h"

namespace {
using namespace ibh;

// Four floats at any multiple of 4 bytes: rows of odd length start there, and
// a global load or store of four dwords needs no more.
typedef float f4_t __attribute__((ext_vector_type(4), aligned(4)));
// Four codes at any byte.
typedef uint32_t u1_t __attribute__((aligned(1)));

struct NormArgs {
    float *y, *s, *h;
    int8_t* q;
    const float *x, *delta, *weight;
    float eps;
    int N, G;                                            // G groups of 128 columns
    size_t xs, ds;                                       // floats between rows of x and delta
};

__device__ __forceinline__ f4_t load4(const float* p, int j, int N) {
    f4_t v = {0.f, 0.f, 0.f, 0.f};
    if (j + 4 <= N) return *(const f4_t*)(p + j);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (j + i < N) v[i] = p[j + i];
    return v;
}
__device__ __forceinline__ void store4(float* p, int j, int N, f4_t v) {
    if (j + 4 <= N) {
        *(f4_t*)(p + j) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (j + i < N) p[j + i] = v[i];
}

// v of the lane that CTRL names, both halves of a double.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)b, CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    v += dpp_f64<0xB1>(v);                               // lane ^ 1
    v += dpp_f64<0x4E>(v);                               // lane ^ 2
    v += dpp_f64<0x124>(v);                              // row_ror 4
    v += dpp_f64<0x128>(v);                              // row_ror 8
    return (lane_f64(v, 0) + lane_f64(v, 16)) + (lane_f64(v, 32) + lane_f64(v, 48));
}

// The largest of 16 lanes, in all of them.
__device__ __forceinline__ uint32_t row_umax(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, false));
}

// 1 / sqrt(a) to about 2^-44: the instruction gives 2^-23 or better, a Newton
// step squares its error.  NaN for a of 0, an infinity or NaN.
__device__ __forceinline__ double rsqrt_f64(double a) {
    const double y = __builtin_amdgcn_rsq(a);
    return __builtin_fma(y * 0.5, __builtin_fma(-a * y, y, 1.0), y);
}
// 1 / a to about 2^-51, likewise with two steps.
__device__ __forceinline__ double rcp_f64(double a) {
    double y = __builtin_amdgcn_rcp(a);
    y = __builtin_fma(__builtin_fma(-a, y, 1.0), y, y);
    return __builtin_fma(__builtin_fma(-a, y, 1.0), y, y);
}

// The sum over the block's wavefronts, the same bits in every thread.
template <int T>
__device__ __forceinline__ double block_sum(double v, double* part) {
    v = wave_sum_f64(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = part[0];
#pragma unroll
    for (int i = 1; i < T / 64; i++) s += part[i];
    return s;
}

// Columns j .. j + 3 of a row.  p = h * weight (rounded), y = p * r, r in 64
// bits (beside subnormal numbers it is beyond fp32).  A code is
// 127 p / max|p| of its 128 columns: r cancels, so codes do not depend on how
// the squares were summed.  In lowest terms a quotient lies 2^-33 or more from
// a border that it does not hit (p and max|p| have 24 bits, and the lowest
// border is max|p| / 254, 8 bits down), the product here is within 2^-43: with
// 2^-38 added before the fraction is cut off, halves go away from zero and
// nothing else changes sides.
__device__ __forceinline__ void emit4(const NormArgs& a, size_t row, int j, f4_t p, double r) {
    if (a.y) {
        f4_t y;
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = (float)((double)p[i] * r);
        store4(a.y + row * a.N, j, a.N, y);
    }
    if (!a.q) return;
    uint32_t bits = 0;                                   // of the largest |p|: as whole numbers a NaN is above all
#pragma unroll
    for (int i = 0; i < 4; i++) bits = max(bits, __float_as_uint(p[i]) & 0x7fffffffu);
    bits = row_umax(bits);
    bits = max(bits, (uint32_t)__shfl_xor((int)bits, 16, 32));   // 32 lanes hold a group
    const float m = __builtin_bit_cast(float, bits);
    const double top = (double)m * r;
    const bool sound = bits < 0x7f800000u && top == top, zero = !sound || top < 1e-10;
    if (j >= a.N) return;
    if ((j & 127) == 0) a.s[row * a.G + j / 128] = !sound ? __builtin_nanf("") : zero ? 1e-10f : (float)(top * (1.0 / 127.0));
    const double k = 127.0 * rcp_f64((double)m);
    uint32_t packed = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const double t = __builtin_fma((double)fabsf(p[i]), k, 0.5 + 0x1p-38);
        const int c = zero ? 0 : (int)t;
        packed |= (uint32_t)((p[i] < 0 ? -c : c) & 255) << (8 * i);
    }
    int8_t* q = a.q + row * a.N;
    if (j + 4 <= a.N) {
        *(u1_t*)(q + j) = packed;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (j + i < a.N) q[j + i] = (int8_t)(packed >> (8 * i));
}

// A row in the registers of a block of T threads, E quads each: x and delta are
// read once, the squares summed in 64 bits (a square of a float cannot overflow
// there), the outputs written from the registers.
template <int T, int E>
__global__ __launch_bounds__(T) void norm_row_kernel(NormArgs a) {
    __shared__ double part[T / 64];
    const size_t row = blockIdx.x;
    const float* x = a.x + row * a.xs;
    f4_t h[E], w[E];
#pragma unroll
    for (int e = 0; e < E; e++) h[e] = load4(x, (e * T + threadIdx.x) * 4, a.N);
    if (a.delta) {
        const float* d = a.delta + row * a.ds;
        f4_t v[E];
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = load4(d, (e * T + threadIdx.x) * 4, a.N);
#pragma unroll
        for (int e = 0; e < E; e++) h[e] += v[e];
    }
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = load4(a.weight, (e * T + threadIdx.x) * 4, a.N);
    double sum = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (a.h) store4(a.h + row * a.N, (e * T + threadIdx.x) * 4, a.N, h[e]);
#pragma unroll
        for (int i = 0; i < 4; i++) sum = __builtin_fma((double)h[e][i], (double)h[e][i], sum);
    }
    const double r = rsqrt_f64(block_sum<T>(sum, part) / a.N + (double)a.eps);
#pragma unroll
    for (int e = 0; e < E; e++) emit4(a, row, (e * T + threadIdx.x) * 4, h[e] * w[e], r);
}

// Rows longer than the registers hold: read twice, the second time from h
// where it is written (each thread reads what it wrote itself).
__global__ __launch_bounds__(1024) void norm_long_kernel(NormArgs a) {
    __shared__ double part[16];
    const size_t row = blockIdx.x;
    const float *x = a.x + row * a.xs, *d = a.delta ? a.delta + row * a.ds : nullptr;
    float* h = a.h ? a.h + row * a.N : nullptr;
    double sum = 0;
    for (int j = threadIdx.x * 4; j < a.N; j += 4096) {
        f4_t v = load4(x, j, a.N);
        if (d) v += load4(d, j, a.N);
        if (h) store4(h, j, a.N, v);
#pragma unroll
        for (int i = 0; i < 4; i++) sum = __builtin_fma((double)v[i], (double)v[i], sum);
    }
    const double r = rsqrt_f64(block_sum<1024>(sum, part) / a.N + (double)a.eps);
    // whole blocks of columns, so that all lanes of a group are there for its maximum
    for (int base = 0; base < a.N; base += 4096) {
        const int j = base + threadIdx.x * 4;
        f4_t v = load4(h ? h : x, j, a.N);
        if (d && !h) v += load4(d, j, a.N);
        emit4(a, row, j, v * load4(a.weight, j, a.N), r);
    }
}

template <int T, int E>
void launch(const NormArgs& a, int B, hipStream_t st) {
    norm_row_kernel<T, E><<<B, T, 0, st>>>(a);
}

}  // namespace

extern "C" int ibh_add_rmsnorm(float* y, int8_t* q, float* s, float* h, const float* x, const float* delta,
                               const float* weight, float eps, int N, int B, int x_stride, int delta_stride,
                               void* stream) {
    if (B == 0) return IBH_OK;
    if (!x || !weight || (!y && !q) || !q != !s || N <= 0 || N > (1 << 30) || B < 0 ||
        (B > 1 && (x_stride < N || (delta && delta_stride < N)))) {
        ibh_set_error("ibh_add_rmsnorm: invalid arguments (N=%d B=%d x_stride=%d delta_stride=%d; x, weight, and y or "
                      "q with s)", N, B, x_stride, delta_stride);
        return IBH_ERROR_PARAM;
    }
    if (!(eps >= 0.f) || !(eps <= 3.4028234e38f)) {
        ibh_set_error("ibh_add_rmsnorm: eps must be a finite number, not negative");
        return IBH_ERROR_PARAM;
    }
    const int G = (N + 127) / 128;
    const size_t rows = (size_t)B * N * 4, xb = ((size_t)(B - 1) * x_stride + N) * 4;
    const size_t db = ((size_t)(B - 1) * delta_stride + N) * 4;
    const struct { const void* p; size_t n; } outs[] = {{y, rows}, {h, rows}, {q, rows / 4}, {s, (size_t)B * G * 4}};
    for (int i = 0; i < 4; i++) {
        // y or h may take the place of x or delta: a thread reads its columns before it writes them
        const bool xin = i < 2 && outs[i].p == x && (B == 1 || x_stride == N);
        const bool din = i < 2 && outs[i].p == delta && (B == 1 || delta_stride == N);
        bool bad = (!xin && ibh_overlap(outs[i].p, outs[i].n, x, xb)) || (!din && ibh_overlap(outs[i].p, outs[i].n, delta, db)) ||
                   ibh_overlap(outs[i].p, outs[i].n, weight, (size_t)N * 4);
        for (int k = 0; k < i; k++) bad |= ibh_overlap(outs[i].p, outs[i].n, outs[k].p, outs[k].n);
        if (bad) {
            ibh_set_error("ibh_add_rmsnorm: an output overlaps another operand");
            return IBH_ERROR_PARAM;
        }
    }
    if (B >= (1 << 22)) {                                // a launch takes less than 2^32 threads
        ibh_set_error("ibh_add_rmsnorm: %d rows are more than one launch takes", B);
        return IBH_ERROR_PARAM;
    }
    const NormArgs a{y, s, h, q, x, delta, weight, eps, N, G, (size_t)x_stride, (size_t)delta_stride};
    hipStream_t st = ibh_resolve_stream(stream);
    // Threads by quads of columns, all in us of the kernel: the fewest that hold the
    // row for short rows (6000 x 200 in 64 threads 5.9, in 256 9.5; 4000 x 1000 in
    // 128 11.1, in 256 13.1); then, for few rows, wide blocks, whose loads are all
    // under way sooner (1 x 4096 in 512 threads 2.8, in 256 3.8; 64 rows 3.9 and 4.8;
    // 512 rows 8.0 and 8.4), for many small ones, of which a CU holds more (1024 rows
    // 10.9 in both, 1500 15.5 and 14.7, 4099 44.6 and 43.2; 4099 x 2048 in 512 22.9, in
    // 64 21.3; 8192 columns in 1024 and 512: 64 rows 4.4 and 4.5, 1024 24.1 and 22.2,
    // 2000 46.7 and 42.8).
    const bool few = B <= 1024;
    if (N <= 256) launch<64, 1>(a, B, st);
    else if (N <= 1024) launch<128, 2>(a, B, st);
    else if (N <= 2048) few ? launch<512, 1>(a, B, st) : launch<64, 8>(a, B, st);
    else if (N <= 4096) few ? launch<512, 2>(a, B, st) : launch<256, 4>(a, B, st);
    else if (N <= 8192) few ? launch<1024, 2>(a, B, st) : launch<512, 4>(a, B, st);
    else if (N <= 16384) launch<1024, 4>(a, B, st);
    else norm_long_kernel<<<B, 1024, 0, st>>>(a);
    IBH_CHECK_LAUNCH("ibh_add_rmsnorm");
    return IBH_OK;
}
