// ibh_lora.hip -- low-rank adapters of many requests beside a shared
// projection: out[b] = base[b] + scale * B (A x[b]) with the adapter of row b.
//
// Two products in a row, the first into t = scale * A x (a few numbers a row),
// so two launches, or one where A is small enough to be read again.  Every byte
// of x, base and out and of each adapter that some row has is needed once: memory
// bounds both.  Sums are fp32 of exact products: up to kFew rows on the vector
// units, beyond on the bf16 matrix cores, where an fp32 number is three bf16
// numbers (8 + 8 + 8 bits, exactly) and an fp16 one two.
#include "ibh_common.h"

namespace {
using namespace ibh;

__device__ unsigned int ibh_lora_err;

constexpr int kFew = 64;            // rows up to which a wavefront holds all ids, one a lane
constexpr int kMaxAdapters = 4096;  // counters of the plan's block
constexpr int kTile = 32;           // rows of one adapter that a block of the matrix kernels takes
constexpr int kStep = 64;           // columns of x that a wavefront takes at a time
constexpr int kOut = 2;             // outputs of a lane group in the second product of few rows
constexpr int kBoth = 512;          // threads that do both products of few rows,
constexpr int kBothOut = 4;         // the outputs of a lane group there,
constexpr int kBothRank = 32;       // and the rank
constexpr size_t kBothMost = 65536; // and numbers of an adapter's a up to which they do
constexpr int kSpan = 256;          // outputs that a block of the second product takes

typedef float f4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4h_t __attribute__((ext_vector_type(4), aligned(2)));

struct Lora {
    const uint16_t *a, *b;
    const float* scales;
    const int32_t* ranks;
    int n, R, N, M;
    float* out;
    const float *base, *x;
    const int32_t* ids;
    int B;
    size_t os, bs, xs;
    float* t;                       // [split][B][Rp]: scale * A x of each row; zeros behind its adapter's rank
    int Rp;                         // R in whole eights
    int S;                          // splits
    struct Tile* tiles;
    int max_tiles;
    const uint16_t *a_end, *b_end;  // behind the arrays
    const float *x_end, *base_end;
};
// Rows of one adapter.  All that a block has to know in one place, so that it
// waits for memory once before its first row.
struct __align__(16) Tile {
    int32_t id, rank, count;        // rank -1: not in the table, 0: no adapter; count 0: no tile
    float scale;
    int32_t row[kTile];
};

template <int KIND>
__device__ __forceinline__ float widen(uint32_t h) {    // of the low half
    if constexpr (KIND == IBH_F16) return f16_to_f32((uint16_t)h);
    else return __uint_as_float(h << 16);
}
// The rank of adapter `id`: 0 for none, -1 where the table does not have it.
__device__ __forceinline__ int rank_of(const Lora& l, int id) {
    if (id < 0) return 0;
    if (id >= l.n) return -1;
    const int r = l.ranks ? l.ranks[id] : l.R;
    return r < 0 || r > l.R ? -1 : r;
}
// Loads from place j of a row of n, zeros behind n.  WHOLE: n is a multiple of
// what is loaded.  Otherwise what lies behind the row is read with it and
// masked, one by one only where the array ends (`end`): every line of code that a
// small launch runs through is one more wait for memory.
template <bool WHOLE>
__device__ __forceinline__ f4_t load4(const float* p, int j, int n, const float* end) {
    f4_t v = {0.f, 0.f, 0.f, 0.f};
    if (j >= n) return v;
    if (WHOLE || p + j + 4 <= end) v = *(const f4_t*)(p + j);
    else
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (p + j + i < end) v[i] = p[j + i];
    if constexpr (!WHOLE)
#pragma unroll
        for (int i = 1; i < 4; i++) v[i] = j + i < n ? v[i] : 0.f;
    return v;
}
template <bool WHOLE>
__device__ __forceinline__ void store4(float* p, int j, int n, f4_t v) {
    if (WHOLE ? j < n : j + 4 <= n) {
        *(f4_t*)(p + j) = v;
        return;
    }
    if constexpr (WHOLE) return;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (j + i < n) p[j + i] = v[i];
}
// Eight 16-bit numbers, likewise.
template <bool WHOLE>
__device__ __forceinline__ u4_t load8h(const uint16_t* p, int j, int n, const uint16_t* end) {
    u4_t v = {0, 0, 0, 0};
    if (j >= n) return v;
    if (WHOLE || p + j + 8 <= end) v = *(const u4h_t*)(p + j);
    else
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (p + j + i < end) v[i / 2] |= (uint32_t)p[j + i] << (16 * (i % 2));
    if (!WHOLE && j + 8 > n)
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] &= (j + 2 * i < n ? 0xffffu : 0) | (j + 2 * i + 1 < n ? 0xffff0000u : 0);
    return v;
}
// Numbers j .. j + 7 of a row of b, zeros from `rank` on.  WHOLE: the row is
// whole eights, so all of them may be read.
template <bool WHOLE>
__device__ __forceinline__ u4_t load_rank(const Lora& l, const uint16_t* p, int j, int rank) {
    if constexpr (!WHOLE) return load8h<false>(p, j, rank, l.b_end);
    u4_t v = {0, 0, 0, 0};
    if (j < rank) v = *(const u4h_t*)(p + j);
    if (rank % 8 && j + 8 > rank)                        // j is a multiple of 8
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] &= (j + 2 * i < rank ? 0xffffu : 0) | (j + 2 * i + 1 < rank ? 0xffff0000u : 0);
    return v;
}

// ── up to kFew rows ──────────────────────────────────────────────────────────
// Each block belongs to a row.  The rows of its adapter are served four at a time
// by the blocks of its first, fifth, ... row: what they share is read from
// memory once and from L2 by the others.  A chain of waits bounds these: ids, an
// adapter's rank, its numbers and x, sums over the block (32 rows of 4096, each
// with an adapter of rank 16: 8.4 MB in 4.1 and 3.2 us, 7.3 in one launch).
struct Few {
    int id, rank, rows;             // rows 0: this block has nothing to do
    // Four numbers, all of them read to pick one: one of an array, or one of four
    // places in the struct, would put it all into LDS, at a place read off the
    // dispatch packet in host memory (10 us for 512 blocks).
    int r0, r1, r2, r3;
    __device__ __forceinline__ int row(int i) const {
        return (r0 & -(i == 0)) | (r1 & -(i == 1)) | (r2 & -(i == 2)) | (r3 & -(i == 3));
    }
};
__device__ __forceinline__ Few few_of(const Lora& l, int me) {
    const int lane = threadIdx.x & 63;
    const int mine = lane < l.B ? max(l.ids[lane], -1) : -2;
    Few f;
    f.id = __builtin_amdgcn_readlane(mine, me);
    f.rank = rank_of(l, f.id);
    uint64_t same = __ballot(mine == f.id);
    f.rows = 0;
    const int before = __popcll(same & ((1ull << me) - 1));
    if (before % 4) return f;
    same &= ~0ull << me;
    f.rows = min(4, __popcll(same));
    auto next = [&] {
        const int r = same ? __ffsll((unsigned long long)same) - 1 : me;
        same &= same - 1;
        return r;
    };
    f.r0 = next(), f.r1 = next(), f.r2 = next(), f.r3 = next();
    return f;
}

// The wavefront's sums of K numbers (2 .. 32): each step gives half of them away
// to the lane across and takes the other half's, 32 exchanges for 32 numbers where
// one sum after the other would take 32 times six.  Returns whose sum a[0] is
// then, -1 in the lanes that hold copies.
template <int K>
__device__ __forceinline__ int wave_sums(float* a) {
    const int lane = threadIdx.x & 63;
    auto across = [](float v, int s) {
        const int b = (int)__float_as_uint(v);
        return s == 0 ? __uint_as_float(__builtin_amdgcn_mov_dpp(b, 0xB1, 0xF, 0xF, false)) :     // lane ^ 1
               s == 1 ? __uint_as_float(__builtin_amdgcn_mov_dpp(b, 0x4E, 0xF, 0xF, false)) :     // lane ^ 2
               s == 2 ? __uint_as_float(__builtin_amdgcn_mov_dpp(b, 0x128, 0xF, 0xF, false)) :    // lane ^ 8
                        __shfl_xor(v, s == 3 ? 16 : s == 4 ? 32 : 4, kWave);
    };
    constexpr int bit[6] = {1, 2, 8, 16, 32, 4};
    int index = 0, copy = 0;
#pragma unroll
    for (int s = 0; s < 6; s++) {
        const int half = K >> (s + 1);
        const uint32_t up = lane & bit[s] ? ~0u : 0u;    // a mask: picked by one, the numbers would go to memory
        if (half) {
#pragma unroll
            for (int i = 0; i < half; i++) {
                const uint32_t x = __float_as_uint(a[i]), y = __float_as_uint(a[i + half]);
                a[i] = __uint_as_float((y & up) | (x & ~up)) + across(__uint_as_float((x & up) | (y & ~up)), s);
            }
            index += half & up;
        } else {
            a[0] += across(a[0], s);
            copy |= up;
        }
    }
    return copy ? -1 : index;
}

// RR ranks of an adapter times NR rows by T threads, which take eights of
// columns; to t, rows Rp apart, zeros behind the adapter's rank.
template <int KIND, bool WHOLE, int T, int RR, int NR, class Store>
__device__ __forceinline__ void shrink_rows(const Lora& l, const Few& f, int r0, float (*part)[T / 64], Store&& store) {
    const int tid = threadIdx.x;
    const uint16_t* a = l.a + ((size_t)f.id * l.R + r0) * l.N;
    const int nr = min(RR, f.rank - r0);
    float acc[RR][NR];
#pragma unroll
    for (int r = 0; r < RR; r++)
#pragma unroll
        for (int i = 0; i < NR; i++) acc[r][i] = 0.f;
    for (int j = tid * 8; j < l.N; j += T * 8) {
        u4_t w[RR];
        f4_t v[NR][2];
#pragma unroll
        for (int r = 0; r < RR; r++) w[r] = r < nr ? load8h<WHOLE>(a + (size_t)r * l.N, j, l.N, l.a_end) : u4_t{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NR; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) v[i][h] = load4<WHOLE>(l.x + f.row(i) * l.xs, j + 4 * h, l.N, l.x_end);
#pragma unroll
        for (int r = 0; r < RR; r++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float we = widen<KIND>(e % 2 ? w[r][e / 2] >> 16 : w[r][e / 2] & 0xffffu);
#pragma unroll
                for (int i = 0; i < NR; i++) acc[r][i] = fmaf(we, v[i][e / 4][e % 4], acc[r][i]);
            }
    }
    const int at = wave_sums<RR * NR>(&acc[0][0]);
    if (at >= 0) part[at][tid >> 6] = acc[0][0];
    __syncthreads();
    if (tid < RR * NR) {
        const int r = tid / NR, i = tid % NR;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < T / 64; w++) s += part[tid][w];
        if (i < f.rows && r0 + r < l.Rp) store(i, r0 + r, r < nr ? s * (l.scales ? l.scales[f.id] : 1.f) : 0.f);
    }
}

template <int KIND, bool WHOLE>
__global__ __launch_bounds__(256) void lora_shrink_few(Lora l) {
    __shared__ float part[16][4];
    const Few f = few_of(l, blockIdx.x);
    const int r0 = blockIdx.y * 4;
    if (!f.rows || f.rank <= 0 || r0 >= (f.rank + 7) / 8 * 8) return;
    auto store = [&](int i, int r, float v) { l.t[(size_t)f.row(i) * l.Rp + r] = v; };
    if (f.rows == 1) shrink_rows<KIND, WHOLE, 256, 4, 1>(l, f, r0, part, store);
    else if (f.rows == 2) shrink_rows<KIND, WHOLE, 256, 4, 2>(l, f, r0, part, store);
    else shrink_rows<KIND, WHOLE, 256, 4, 4>(l, f, r0, part, store);
}

// Outputs of block `block` of a row: a row of b in `1 << lg` lanes, eight numbers
// each; OUT outputs a lane group.
template <int KIND, bool WHOLE, int T, int OUT, int NR>
struct Expand {
    u4_t w[OUT];
    float y[OUT][NR];
    int sub, per, m0, lg;

    // what does not need t
    __device__ __forceinline__ Expand(const Lora& l, const Few& f, int lg_, int block) : lg(lg_) {
        sub = threadIdx.x & ((1 << lg) - 1), per = T >> lg;
        m0 = block * per * OUT + (threadIdx.x >> lg);
        const uint16_t* b = l.b + (size_t)f.id * l.M * l.R;
#pragma unroll
        for (int o = 0; o < OUT; o++) {
            const int m = m0 + o * per;
            w[o] = m < l.M ? load_rank<WHOLE>(l, b + (size_t)m * l.R, 8 * sub, f.rank) : u4_t{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < NR; i++) y[o][i] = l.base && sub == 0 && m < l.M ? l.base[f.row(i) * l.bs + m] : 0.f;
        }
    }
    template <class Load>
    __device__ __forceinline__ void finish(const Lora& l, const Few& f, Load&& load) const {
        f4_t t[NR][2];
#pragma unroll
        for (int i = 0; i < NR; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) t[i][h] = 8 * sub < f.rank ? load(i, 8 * sub + 4 * h) : f4_t{0.f, 0.f, 0.f, 0.f};
        float s[OUT][NR];
#pragma unroll
        for (int o = 0; o < OUT; o++) {
#pragma unroll
            for (int i = 0; i < NR; i++) s[o][i] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float we = widen<KIND>(e % 2 ? w[o][e / 2] >> 16 : w[o][e / 2] & 0xffffu);
#pragma unroll
                for (int i = 0; i < NR; i++) s[o][i] = fmaf(we, t[i][e / 4][e % 4], s[o][i]);
            }
        }
        for (int k = 0; k < lg; k++)                     // the lanes of an output, all outputs side by side
#pragma unroll
            for (int o = 0; o < OUT; o++)
#pragma unroll
                for (int i = 0; i < NR; i++) s[o][i] += __shfl_xor(s[o][i], 1 << k, kWave);
        if (sub) return;
#pragma unroll
        for (int o = 0; o < OUT; o++) {
            const int m = m0 + o * per;
            if (m >= l.M) break;
#pragma unroll
            for (int i = 0; i < NR; i++)
                if (i < f.rows) l.out[f.row(i) * l.os + m] = y[o][i] + s[o][i];
        }
    }
};

// Rows without an adapter: base; with one that is not in the table: NaN.
__device__ __forceinline__ void few_without(const Lora& l, const Few& f, int span, int block) {
    if (f.rank < 0 && threadIdx.x == 0 && block == 0) atomicOr(&ibh_lora_err, IBH_DEVERR_LORA);
    if (f.rank == 0 && l.out == l.base) return;
    const int m0 = block * span;
    for (int i = 0; i < f.rows; i++)
        for (int m = m0 + threadIdx.x; m < min(m0 + span, l.M); m += blockDim.x)
            l.out[f.row(i) * l.os + m] = f.rank < 0 ? __builtin_nanf("") : l.base ? l.base[f.row(i) * l.bs + m] : 0.f;
}

template <int KIND, bool WHOLE, int NR>
__device__ __forceinline__ void expand_rows(const Lora& l, const Few& f, int lg) {
    Expand<KIND, WHOLE, 256, kOut, NR>(l, f, lg, blockIdx.x).finish(l, f, [&](int i, int r) {
        return *(const f4_t*)(l.t + (size_t)f.row(i) * l.Rp + r);
    });
}
// Outputs in the first dimension, rows in the second, which has room for 65535
// blocks: 2^20 outputs in sixteens are one more (64 x 4096, rank 32: 5.6 us, rows
// first 5.8; eight adapters instead of 64: 4.8 and 7.3; 64 x 8192, rank 256: 58
// and 61; 16 x 4096, rank 128: 6.0 and 5.6).
template <int KIND, bool WHOLE>
__global__ __launch_bounds__(256) void lora_expand_few(Lora l, int lg) {
    const Few f = few_of(l, blockIdx.y);
    if (!f.rows) return;
    if (f.rank <= 0) few_without(l, f, (256 >> lg) * kOut, blockIdx.x);
    else if (f.rows == 1) expand_rows<KIND, WHOLE, 1>(l, f, lg);
    else if (f.rows == 2) expand_rows<KIND, WHOLE, 2>(l, f, lg);
    else expand_rows<KIND, WHOLE, 4>(l, f, lg);
}

// Both products in one launch where an adapter's a is small: every block that
// takes outputs of some rows works their t out by itself.  Rows in the first
// dimension: with 8, 16, 24, ... of them a row's blocks come to one XCD, whose L2
// reads a once for all of them (32 x 4096, rank 16: 7.2 us, 8.7 with the outputs
// first); the second has 256 blocks at most.
template <int KIND, bool WHOLE, int NR>
__device__ __forceinline__ void both_rows(const Lora& l, const Few& f, int lg, float (*part)[kBoth / 64], float* t) {
    const Expand<KIND, WHOLE, kBoth, kBothOut, NR> e(l, f, lg, blockIdx.y);
    for (int r0 = 0; r0 < (f.rank + 7) / 8 * 8; r0 += 8) {
        if (r0) __syncthreads();
        shrink_rows<KIND, WHOLE, kBoth, 8, NR>(l, f, r0, part, [&](int i, int r, float v) { t[i * l.Rp + r] = v; });
    }
    __syncthreads();
    e.finish(l, f, [&](int i, int r) { return *(const f4_t*)(t + min(i, f.rows - 1) * l.Rp + r); });
}
template <int KIND, bool WHOLE>
__global__ __launch_bounds__(kBoth) void lora_both_few(Lora l, int lg) {
    __shared__ float part[32][kBoth / 64];
    __shared__ __align__(16) float t[4 * kBothRank];
    const Few f = few_of(l, blockIdx.x);
    if (!f.rows) return;
    if (f.rank <= 0) few_without(l, f, (kBoth >> lg) * kBothOut, blockIdx.y);
    else if (f.rows == 1) both_rows<KIND, WHOLE, 1>(l, f, lg, part, t);
    else if (f.rows == 2) both_rows<KIND, WHOLE, 2>(l, f, lg, part, t);
    else both_rows<KIND, WHOLE, 4>(l, f, lg, part, t);
}

// ── more rows: tiles of one adapter's rows on the matrix cores ───────────────
// One block sorts the rows by adapter (counting; the order within one adapter
// is left to chance and changes no result: a row's sums do not depend on its
// place) and cuts each adapter's rows into tiles.  3.8 us for 120 rows, 6.1 for
// 4099: 1.5 until ids are there, the rest code that is fetched once and LDS
// atomics one behind the other.
__global__ __launch_bounds__(1024) void lora_plan(Lora l) {
    constexpr int kKept = 8;                             // rows of a thread that stay in registers
    __shared__ int32_t count[kMaxAdapters + 2], more[kMaxAdapters + 2];   // the keys' rows: those, the others
    __shared__ int32_t wave_tiles[16];
    const int tid = threadIdx.x, lane = tid & 63, keys = l.n + 2;   // n: no adapter; n + 1: not in the table
    int key[kKept], at[kKept];
#pragma unroll
    for (int u = 0; u < kKept; u++) key[u] = u * 1024 + tid < l.B ? l.ids[u * 1024 + tid] : 0;
    const float scale0 = l.scales && tid < l.n ? l.scales[tid] : 1.f;   // of the first keys, under way with the ids
    for (int i = tid; i < keys; i += 1024) count[i] = more[i] = 0;
    auto key_of = [&](int id) {
        const int rank = rank_of(l, id);
        return rank < 0 ? l.n + 1 : rank == 0 ? l.n : id;
    };
#pragma unroll
    for (int u = 0; u < kKept; u++) key[u] = u * 1024 + tid < l.B ? key_of(key[u]) : -1;
    __syncthreads();
    // adds the wavefront's rows to the counters of their keys, -1 for none, and
    // returns what each row found there: those that share the first row's key
    // (packed prompts: all of them) in one addition
    auto add = [&](int32_t* to, int k) {
        const int first = __builtin_amdgcn_readfirstlane(k);
        const uint64_t same = __ballot(k == first);
        int got = 0;
        if (k != first) {
            if (k >= 0) got = atomicAdd(&to[k], 1);
        } else if (first >= 0) {
            if (lane == 0) got = atomicAdd(&to[first], __popcll(same));
            got = __builtin_amdgcn_readfirstlane(got) + __popcll(same & ((1ull << lane) - 1));
        }
        return got;
    };
    auto later = [&](auto&& f) {                         // whole wavefronts go on together
        for (int i = kKept * 1024 + (tid & ~63); i < l.B; i += 1024) f(i + lane < l.B ? key_of(l.ids[i + lane]) : -1, i + lane);
    };
#pragma unroll
    for (int u = 0; u < kKept; u++)
        if (u * 1024 < l.B) at[u] = add(count, key[u]);
    later([&](int k, int) { add(more, k); });
    __syncthreads();
    // each thread's run of keys: tiles in front of it
    const int per = (keys + 1023) / 1024, k0 = min(tid * per, keys), k1 = min(k0 + per, keys);
    int tiles = 0;
    for (int k = k0; k < k1; k++) tiles += (count[k] + more[k] + kTile - 1) / kTile;
    int it = tiles;
    for (int o = 1; o < 64; o <<= 1) {
        const int p = __shfl_up(it, o, 64);
        if (lane >= o) it += p;
    }
    if (lane == 63) wave_tiles[tid >> 6] = it;
    __syncthreads();
    it -= tiles;
    int all = 0;
    for (int w = 0; w < 16; w++) {
        if (w == tid >> 6) it += all;
        all += wave_tiles[w];
    }
    for (int k = k0; k < k1; k++) {
        const int first = count[k], c = first + more[k];
        if (!c) continue;
        const int rank = k < l.n ? (l.ranks ? l.ranks[k] : l.R) : l.n - k;
        const float scale = k >= l.n || !l.scales ? 1.f : per == 1 ? scale0 : l.scales[k];
        count[k] = it * kTile;                           // from here on: the place of its first row,
        more[k] = it * kTile + first;                    // and of its next one
        for (int j = 0; j < c; j += kTile, it++) *(int4*)&l.tiles[it] = make_int4(k, rank, min(kTile, c - j), __float_as_int(scale));
    }
    for (int i = all + tid; i < l.max_tiles; i += 1024) l.tiles[i].count = 0;
    __syncthreads();
    auto place = [&](int k, int row, int i) {
        if (k >= 0) l.tiles[i / kTile].row[i % kTile] = row;
    };
#pragma unroll
    for (int u = 0; u < kKept; u++)
        if (u * 1024 < l.B) place(key[u], u * 1024 + tid, key[u] >= 0 ? count[key[u]] + at[u] : 0);
    later([&](int k, int row) {
        const int i = add(more, k);
        place(k, row, i);
    });
}

// fp32 numbers as bf16 numbers, upper halves cut off one after the other: 8
// bits each, all 24 in three.  Nothing is lost of numbers of 2^-110 and more; of
// smaller ones what lies below 2^-133, the last place of a bf16 number (the matrix
// cores take subnormal ones as they are).  An infinity leaves NaN below it: a sum
// that holds one becomes NaN, as it does beside the next one of the other sign.
__device__ __forceinline__ uint32_t upper(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
}
__device__ __forceinline__ float below(float v) {
    return v - __uint_as_float(__float_as_uint(v) & 0xffff0000u);
}
// Eight 16-bit numbers of an adapter as bf16: one piece, or two for fp16 (8 and
// 3 bits).
template <int KIND>
__device__ __forceinline__ void pieces(u4_t v, v8bf* p) {
    if constexpr (KIND == IBH_BF16) p[0] = __builtin_bit_cast(v8bf, v);
    else {
        u4_t hi, lo;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float a = f16_to_f32((uint16_t)v[i]), b = f16_to_f32((uint16_t)(v[i] >> 16));
            hi[i] = upper(a, b);
            lo[i] = upper(below(a), below(b));
        }
        p[0] = __builtin_bit_cast(v8bf, hi);
        p[1] = __builtin_bit_cast(v8bf, lo);
    }
}

// t of a tile of rows and RT * 16 ranks over a share of the columns.  Each
// wavefront takes 64 columns of all rows at a time, the next 64 under way: every
// number of x is loaded, cut into pieces and multiplied by one lane, straight in
// the matrix instructions' own order (16 rows, 32 columns in eights).  4099 x
// 4096: 17 us with rank 16 in bf16 (4.1 TB/s), 22 with rank 32 in fp16, whose
// pieces take half of the vector instructions; 26 with the pieces in LDS.
template <int KIND, bool WHOLE, int RT>
__global__ __launch_bounds__(256, RT <= 2 ? 3 : 2) void lora_shrink_tile(Lora l) {
    constexpr int P = KIND == IBH_F16 ? 2 : 1;
    __shared__ v4f join[4][2 * RT][64];
    const Tile& tl = l.tiles[blockIdx.y];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane % 16, q = lane / 16;
    const int row[2] = {tl.row[c], tl.row[16 + c]};
    const int id = tl.id, rank = tl.rank, count = tl.count, r0 = blockIdx.z * RT * 16;
    const float scale = tl.scale;
    if (!count || r0 >= (rank + 7) / 8 * 8) return;
    const int steps = (l.N + kStep - 1) / kStep;
    const int s0 = (int)((int64_t)steps * blockIdx.x / l.S), s1 = (int)((int64_t)steps * (blockIdx.x + 1) / l.S);
    // Places of the tile without a row, and ranks that the adapter has not, load
    // another's: what comes of them is not stored.
    const float* xp[2];
    const uint16_t* ap[RT];
#pragma unroll
    for (int h = 0; h < 2; h++) xp[h] = l.x + (h * 16 + c < count ? row[h] : tl.row[0]) * l.xs;
#pragma unroll
    for (int i = 0; i < RT; i++) ap[i] = l.a + ((size_t)id * l.R + min(r0 + i * 16 + c, rank - 1)) * l.N;
    struct Piece {
        f4_t x[2][2][2];
        u4_t a[RT][2];
    };
    auto fetch = [&](int s, Piece& p) {
        const int k0 = s * kStep + q * 8;
#pragma unroll
        for (int k = 0; k < 2; k++) {
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 2; e++) p.x[h][k][e] = load4<WHOLE>(xp[h], k0 + 32 * k + 4 * e, l.N, l.x_end);
#pragma unroll
            for (int i = 0; i < RT; i++) p.a[i][k] = load8h<WHOLE>(ap[i], k0 + 32 * k, l.N, l.a_end);
        }
    };
    v4f acc[2][RT];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < RT; i++) acc[h][i] = v4f{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Piece& p) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            v8bf ba[RT][2];
#pragma unroll
            for (int i = 0; i < RT; i++) pieces<KIND>(p.a[i][k], ba[i]);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = p.x[h][k][e / 4][e % 4];
#pragma unroll
                for (int w = 0; w < 3; w++) {
                    u4_t u;
#pragma unroll
                    for (int e = 0; e < 4; e++) u[e] = upper(v[2 * e], v[2 * e + 1]);
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = below(v[e]);
#pragma unroll
                    for (int i = 0; i < RT; i++)
#pragma unroll
                        for (int j = 0; j < P; j++)
                            acc[h][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ba[i][j], __builtin_bit_cast(v8bf, u), acc[h][i], 0, 0, 0);
                }
            }
        }
    };
    Piece p0, p1;
    int s = s0 + wave;
    if (s < s1) fetch(s, p0);
    if (s + 4 < s1) fetch(s + 4, p1);
    for (; s < s1; s += 8) {
        multiply(p0);
        if (s + 8 < s1) fetch(s + 8, p0);
        if (s + 4 < s1) multiply(p1);
        if (s + 12 < s1) fetch(s + 12, p1);
    }
    // the wavefronts' sums join; lane: row lane % 16 of 16, ranks lane / 16 * 4 .. + 3
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < RT; i++) join[wave][h * RT + i][lane] = acc[h][i];
    lds_barrier();
    for (int w = wave; w < 2 * RT; w += 4) {
        const int at = w / RT * 16 + c, r = r0 + w % RT * 16 + q * 4;
        v4f v = ((join[0][w][lane] + join[1][w][lane]) + (join[2][w][lane] + join[3][w][lane])) * scale;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = r + e < rank ? v[e] : 0.f;
        if (at < count && r < l.Rp) *(v4f*)(l.t + ((size_t)blockIdx.x * l.B + tl.row[at]) * l.Rp + r) = v;
    }
}

// out of a tile of rows and kSpan outputs.  t's splits are added up and cut
// into pieces in LDS.  A wavefront multiplies 64 outputs of all rows, four
// matrix tiles beside each other (tile j holds outputs 4 c + j, so that a lane
// has four neighbours); through LDS they come to wavefronts that add 256
// outputs of a row to base at once, whole kilobytes of memory.  Neighbouring
// blocks take neighbouring outputs: 4099 x 4096 of rank 32 take 32 us, where plain
// copies take 26 in this order and 36 with a block's outputs one after the other.
template <int KIND, bool WHOLE>
__global__ __launch_bounds__(256, 3) void lora_expand_tile(Lora l) {
    constexpr int P = KIND == IBH_F16 ? 2 : 1;
    extern __shared__ __align__(16) uint16_t st[];       // t [3][kTile][kr], then, in its place, outputs
    float (*so)[kSpan + 4] = (float (*)[kSpan + 4])st;
    const Tile& tl = l.tiles[blockIdx.y];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane % 16, q = lane / 16;
    const int id = tl.id, rank = tl.rank, count = tl.count, m0 = blockIdx.x * kSpan;
    size_t row[8];                                       // this wavefront's to add and store
#pragma unroll
    for (int i = 0; i < 8; i++) row[i] = tl.row[wave * 8 + i];
    const int mine = min(8, count - wave * 8);
    if (!count) return;
    if (rank < 0 && tid == 0 && blockIdx.x == 0) atomicOr(&ibh_lora_err, IBH_DEVERR_LORA);
    if (rank == 0 && l.out == l.base) return;
    f4_t y[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        y[i] = l.base && i < mine ? load4<WHOLE>(l.base + row[i] * l.bs, m0 + 4 * lane, l.M, l.base_end) : f4_t{0.f, 0.f, 0.f, 0.f};
    if (rank <= 0) {                                     // no adapter: base; not in the table: NaN
        const float nan = __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < mine) store4<WHOLE>(l.out + row[i] * l.os, m0 + 4 * lane, l.M, rank < 0 ? f4_t{nan, nan, nan, nan} : y[i]);
        return;
    }
    const uint16_t* b[4];
#pragma unroll
    for (int j = 0; j < 4; j++) b[j] = l.b + ((size_t)id * l.M + min(m0 + wave * 64 + 4 * c + j, l.M - 1)) * l.R;
    u4_t w[4];
    auto fetch = [&](int k) {
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = load_rank<WHOLE>(l, b[j], k * 32 + q * 8, rank);
    };
    fetch(0);
    const int ks = (rank + 31) / 32, kr = ks * 32 + 8;
    for (int i = tid; i < kTile * ks * 8; i += 256) {
        const int k = i / (ks * 8), r = i % (ks * 8) * 4;
        v4f v = {0.f, 0.f, 0.f, 0.f};
        if (k < count && r < (rank + 7) / 8 * 8) {
            const float* t = l.t + (size_t)tl.row[k] * l.Rp + r;
#pragma unroll 8
            for (int s = 0; s < l.S; s++) v += *(const v4f*)(t + (size_t)s * l.B * l.Rp);
        }
        float e[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int p = 0; p < 3; p++) {
            *(uint2*)&st[(p * kTile + k) * kr + r] = make_uint2(upper(e[0], e[1]), upper(e[2], e[3]));
#pragma unroll
            for (int u = 0; u < 4; u++) e[u] = below(e[u]);
        }
    }
    lds_barrier();
    v4f acc[2][4];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[h][j] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < ks; k++) {
        v8bf at[2][3];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int p = 0; p < 3; p++) at[h][p] = *(const v8bf*)&st[(p * kTile + h * 16 + c) * kr + k * 32 + q * 8];
        u4_t now[4];
#pragma unroll
        for (int j = 0; j < 4; j++) now[j] = w[j];
        if (k + 1 < ks) fetch(k + 1);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v8bf bw[2];
            pieces<KIND>(now[j], bw);
#pragma unroll
            for (int i = 0; i < P; i++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int p = 0; p < 3; p++)
                        acc[h][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at[h][p], bw[i], acc[h][j], 0, 0, 0);
        }
    }
    lds_barrier();
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            *(v4f*)&so[h * 16 + 4 * q + i][wave * 64 + 4 * c] = v4f{acc[h][0][i], acc[h][1][i], acc[h][2][i], acc[h][3][i]};
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < mine)
            store4<WHOLE>(l.out + row[i] * l.os, m0 + 4 * lane, l.M, y[i] + *(const f4_t*)&so[wave * 8 + i][4 * lane]);
}

bool adapters_ok(const ibh_lora_adapters* l, const char* who) {
    if (!l || !l->a || !l->b || l->n <= 0 || l->n > kMaxAdapters || l->rank <= 0 || l->rank > IBH_LORA_MAX_RANK || l->N <= 0 || l->M <= 0 ||
        l->N > (1 << 20) || l->M > (1 << 20) || (l->kind != IBH_F16 && l->kind != IBH_BF16)) {
        if (!l) ibh_set_error("%s: no adapters given", who);
        else
            ibh_set_error("%s: invalid adapters (n=%d rank=%d N=%d M=%d kind=%d; up to %d adapters of rank "
                          "up to %d, IBH_F16 or IBH_BF16)",
                          who, l->n, l->rank, l->N, l->M, l->kind, kMaxAdapters, IBH_LORA_MAX_RANK);
        return false;
    }
    return true;
}

// How a call is cut.
struct LoraPlan {
    bool few, both;
    int lg;                                              // lanes of a row of b, their logarithm
    int Rp, S, max_tiles;
    size_t plan_bytes, bytes;
};
LoraPlan plan_of(const ibh_lora_adapters* l, int B) {
    LoraPlan p;
    p.few = B <= kFew;
    p.lg = 0;
    while (8 << p.lg < l->rank) p.lg++;
    // One launch where a is small and a block a CU holds all outputs: it reads a
    // once for each block of outputs, eight ranks after eight, but spares a launch
    // and a workspace, 4 us of an eager call.  Kernels alone, one and two launches, in us:
    //   outputs     1 x 2048, rank 8: 4.4 and 5.5; 32 x 4096, rank 16: 7.3 in both, with
    //               14336 outputs 12.8 and 9.6
    //   numbers     32 rows, rank 16 by 3584, 5120, 6144, 8192: 7.0 and 7.1, 7.9 and 7.8,
    //               8.2 and 8.1, 8.9 in both; one row of 8192: 7.4 and 7.1; 32 rows, rank
    //               32 by 4096: 11.0 and 8.9, rank 8 by 8192: 5.9 and 7.5
    //   rank        32 rows by 65536 numbers, rank 16, 32, 64, 128, 256: 7.3 in both, 8.4
    //               and 7.1, 11.9 and 7.2, 20 and 8.2, 67 and 11
    const int span = (kBoth >> p.lg) * kBothOut;
    p.both = p.few && l->rank <= kBothRank && (size_t)l->rank * l->N <= kBothMost && (size_t)B * ((l->M + span - 1) / span) <= 256;
    p.Rp = (l->rank + 7) / 8 * 8;
    p.S = 1;
    p.max_tiles = 0;
    p.plan_bytes = 0;
    if (!p.few) {
        p.max_tiles = B / kTile + min(l->n + 2, B);
        p.plan_bytes = sizeof(Tile) * (size_t)p.max_tiles;
        // The blocks that share a tile's columns, eights because the second product
        // adds t up eight at a time.  More of them shorten the first product's chain
        // and lengthen the second, the more rows the more (both kernels, eight bf16
        // adapters, 4096 outputs, us): 16 and 8 for 300 x 8192 of rank 32 take 14.0 and
        // 16.9, for 1000 x 8192 of rank 64 28.4 and 26.1, for 300 x 2048 of rank 32 11.4
        // in both; 8 and 1 for 500 x 1024 of rank 32 11.7 and 16.4, for 4099 x 1024 of
        // rank 64 55.3 and 49.7; 8, 4 and 1 for 4099 x 2048 of rank 16 41.1, 42.2 and 43.5;
        // 8 and 10 for 4099 x 5120 of rank 64 74.8 and 80.9.
        p.S = l->N <= B / 4 ? 1 : B <= 512 && l->N > 4096 ? 16 : 8;
    }
    p.bytes = p.both ? 0 : p.plan_bytes + (size_t)p.S * B * p.Rp * 4;
    return p;
}

template <int KIND, bool WHOLE>
void launch_shrink(const Lora& l, const LoraPlan& p, hipStream_t st) {
    const dim3 grid(l.S, l.max_tiles, (l.R + 63) / 64);  // a tile's splits beside each other
    if (p.few) lora_shrink_few<KIND, WHOLE><<<dim3(l.B, (l.Rp + 3) / 4), 256, 0, st>>>(l);
    else if (l.R <= 16) lora_shrink_tile<KIND, WHOLE, 1><<<grid, 256, 0, st>>>(l);
    else if (l.R <= 32) lora_shrink_tile<KIND, WHOLE, 2><<<grid, 256, 0, st>>>(l);
    else lora_shrink_tile<KIND, WHOLE, 4><<<grid, 256, 0, st>>>(l);
}
template <int KIND, bool WHOLE>
void launch_expand(const Lora& l, const LoraPlan& p, int lg, hipStream_t st) {
    const int span = (256 >> lg) * kOut;
    if (p.few) lora_expand_few<KIND, WHOLE><<<dim3((l.M + span - 1) / span, l.B), 256, 0, st>>>(l, lg);
    else
        lora_expand_tile<KIND, WHOLE><<<dim3((l.M + kSpan - 1) / kSpan, l.max_tiles), 256,
                                        max(3 * kTile * ((l.R + 31) / 32 * 32 + 8) * 2, kTile * (kSpan + 4) * 4), st>>>(l);
}
template <int KIND>
int launch(const Lora& l, const LoraPlan& p, hipStream_t st) {
    const int lg = p.lg;
    const bool whole_a = l.N % 8 == 0, whole_b = l.R % 8 == 0 && l.M % 4 == 0;
    if (p.both) {
        const int span = (kBoth >> lg) * kBothOut;
        const dim3 grid(l.B, (l.M + span - 1) / span);
        if (whole_a && whole_b) lora_both_few<KIND, true><<<grid, kBoth, 0, st>>>(l, lg);
        else lora_both_few<KIND, false><<<grid, kBoth, 0, st>>>(l, lg);
        IBH_CHECK_LAUNCH("ibh_lora");
        return IBH_OK;
    }
    if (!p.few) {
        lora_plan<<<1, 1024, 0, st>>>(l);
        IBH_CHECK_LAUNCH("ibh_lora");
    }
    if (whole_a) launch_shrink<KIND, true>(l, p, st);
    else launch_shrink<KIND, false>(l, p, st);
    IBH_CHECK_LAUNCH("ibh_lora");
    if (whole_b) launch_expand<KIND, true>(l, p, lg, st);
    else launch_expand<KIND, false>(l, p, lg, st);
    IBH_CHECK_LAUNCH("ibh_lora");
    return IBH_OK;
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
    return plan_of(l, B).bytes;
}

extern "C" int ibh_lora(const ibh_lora_adapters* l, float* out, const float* base, const float* x, const int32_t* ids,
                        int B, int out_stride, int base_stride, int x_stride, void* ws, size_t ws_bytes, void* stream) {
    if (B == 0) return IBH_OK;
    if (!adapters_ok(l, "ibh_lora")) return IBH_ERROR_PARAM;
    if (!out || !x || !ids || B < 0 || (B > 1 && (out_stride < l->M || (base && base_stride < l->M) || x_stride < l->N))) {
        ibh_set_error("ibh_lora: invalid arguments (B=%d out_stride=%d base_stride=%d x_stride=%d)", B, out_stride,
                      base_stride, x_stride);
        return IBH_ERROR_PARAM;
    }
    const size_t rows = B, ob = ((rows - 1) * out_stride + l->M) * 4, bb = ((rows - 1) * base_stride + l->M) * 4;
    const size_t xb = ((rows - 1) * x_stride + l->N) * 4, n = l->n;
    const size_t om = (size_t)l->M * 4, os = (size_t)out_stride * 4;
    if (ibh_rows_overlap(rows, out, om, os, x, (size_t)l->N * 4, (size_t)x_stride * 4) ||
        (!(out == base && (B == 1 || out_stride == base_stride)) && ibh_rows_overlap(rows, out, om, os, base, om, (size_t)base_stride * 4)) ||
        ibh_overlap(out, ob, ids, rows * 4) || ibh_overlap(out, ob, l->a, n * l->rank * l->N * 2) ||
        ibh_overlap(out, ob, l->b, n * l->rank * l->M * 2) || ibh_overlap(out, ob, l->scales, n * 4) ||
        ibh_overlap(out, ob, l->ranks, n * 4)) {
        ibh_set_error("ibh_lora: out overlaps another operand");
        return IBH_ERROR_PARAM;
    }
    const LoraPlan p = plan_of(l, B);
    // a launch takes less than 2^32 threads, and 65535 tiles in its second dimension
    if (!p.few && (p.max_tiles > 65535 ||
                   (size_t)p.max_tiles * max((l->M + kSpan - 1) / kSpan, p.S * ((l->rank + 63) / 64)) >= (1 << 24))) {
        ibh_set_error("ibh_lora: %d rows are more than one launch takes", B);
        return IBH_ERROR_PARAM;
    }
    uint8_t* w = nullptr;
    if (p.bytes) {
        w = (uint8_t*)(ws ? (ws_bytes >= p.bytes && !((uintptr_t)ws & 15) ? ws : nullptr) : ibh_workspace(p.bytes));
        if (!w) {
            ibh_set_error("ibh_lora: a workspace of %zu bytes on 16 bytes is needed", p.bytes);
            return IBH_ERROR_MEMORY;
        }
    }
    const Lora a{(const uint16_t*)l->a, (const uint16_t*)l->b, l->scales, l->ranks, l->n, l->rank, l->N, l->M, out, base, x,
                 ids, B, (size_t)out_stride, (size_t)base_stride, (size_t)x_stride, (float*)(w + p.plan_bytes), p.Rp, p.S,
                 (Tile*)w, p.max_tiles, (const uint16_t*)l->a + n * l->rank * l->N,
                 (const uint16_t*)l->b + n * l->rank * l->M, x + xb / 4, base ? base + bb / 4 : nullptr};
    hipStream_t st = ibh_resolve_stream(stream);
    return l->kind == IBH_F16 ? launch<IBH_F16>(a, p, st) : launch<IBH_BF16>(a, p, st);
}
