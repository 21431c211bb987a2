// ibh_kv4.hip -- paged 4-bit KV cache of several sequences (gfx950): append,
// read back, attention with accumulated weights, eviction by those weights.
//
// A page holds 64 positions.  For each KV head it is 72 head_dim bytes, one
// after the other:
//   key codes    32 hd  [position / 32][dim / 64][lane 64][position / 16 % 2][8 B]
//   key pairs     4 hd  [dim / 64][slot 64] (scale, mid) fp16
//   value codes  32 hd  [dim / 32][lane 64][dim / 16 % 2][8 B]
//   value pairs   4 hd  [dim / 64][slot 64] (scale, mid) fp16
// Both kinds of codes lie as a wavefront multiplies them (v_mfma_i32_16x16x64
// _i8: lane l holds 16 elements of the summed index, 16 (l / 16) .., of column
// l % 16): a key lane is (position % 16, 16 dims), a value lane (dim % 16, 16
// slots), position t of a page having slot 4 (t % 16) + t / 16.  The 8 bytes
// are two words, byte i of word w the elements 8 w + i (low nibble) and
// 8 w + 4 + i (high), so that two masks turn a word into eight int8 operands.
// An element stands for mid + scale * (code - 8).
#include "ibh_common.h"

#include <type_traits>

using namespace ibh;

namespace {

constexpr int kPage = IBH_KV4_PAGE;
static_assert(kPage == 64, "a page is one MFMA's summed index");

__device__ unsigned int ibh_kv4_err;                     // IBH_DEVERR_* bits of this file's kernels

struct Kv4 {
    uint8_t* pool;
    const int32_t* table;
    int32_t* lens;
    int n_pages, n_seq, max_pages, n_kv, hd;
};

__device__ __forceinline__ void raise_table() {
    __hip_atomic_fetch_or(&ibh_kv4_err, (unsigned)IBH_DEVERR_KV4_TABLE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Read through the scalar cache: no kernel that reads the table or the lengths
// here writes them (kv4_move writes lengths and reads none).
__device__ __forceinline__ int ld_uniform(const int32_t* p) {
    return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
}
// A sequence's length; one outside its table row is cut to it and reported.
__device__ __forceinline__ int seq_len(const Kv4& c, int seq, bool* bad) {
    const int n = ld_uniform(c.lens + seq), cap = c.max_pages * kPage;
    const int m = n < 0 ? 0 : (n > cap ? cap : n);
    *bad = m != n;
    return m;
}
__device__ __forceinline__ const uint8_t* page_by_id(const Kv4& c, int id, int h) {
    if ((unsigned)id >= (unsigned)c.n_pages) return nullptr;
    return c.pool + ((size_t)id * c.n_kv + h) * (size_t)(72 * c.hd);
}
// page_at() where all arguments are the same for the whole wavefront.
__device__ __forceinline__ const uint8_t* page_of_wave(const Kv4& c, int seq, int p, int h) {
    return page_by_id(c, ld_uniform(c.table + (size_t)seq * c.max_pages + p), h);
}
// Head h's part of page p of a sequence, or null where the table names no page of the pool.
__device__ __forceinline__ uint8_t* page_at(const Kv4& c, int seq, int p, int h) {
    const int id = c.table[(size_t)seq * c.max_pages + p];
    if ((unsigned)id >= (unsigned)c.n_pages) return nullptr;
    return c.pool + ((size_t)id * c.n_kv + h) * (size_t)(72 * c.hd);
}

__device__ __forceinline__ float h2f(uint32_t bits) { return f16_to_f32((uint16_t)bits); }
__device__ __forceinline__ uint32_t f2h(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }   // to nearest, ties to even

__device__ __forceinline__ int slot_of(int t) { return 4 * (t & 15) + (t >> 4); }
__device__ __forceinline__ int key_off(int t, int g, int b16, int hdg) {   // 8 bytes: dims 64 g + 16 b16 ..
    return ((t >> 5) * hdg + g) * 1024 + (b16 * 16 + (t & 15)) * 16 + ((t >> 4) & 1) * 8;
}
// The word of value dim d (of the head) that holds positions 16 i + 2 r (low) and 16 i + 2 r + 1 (high) in its byte i.
__device__ __forceinline__ int val_off(int d, int r) {
    return (d >> 5) * 1024 + ((r >> 1) * 16 + (d & 15)) * 16 + ((d >> 4) & 1) * 8 + (r & 1) * 4;
}

// ── append ───────────────────────────────────────────────────────────────────
// Block (64 dims, side, head, page, sequence), 4 threads a position: thread
// (t, cq) holds dims 16 i + 4 cq .. + 3.  The group's ends give scale =
// f16((hi - lo) / 15) and mid = f16(lo + 8 scale).  A code is the quotient (x -
// mid) / scale by the reciprocal, which is at most 2^-19 off (three roundings
// of 2^-24 of at most 9), rounded; where it comes within 2^-17 of a border
// the wavefront compares x - mid with the exact borders (c +- 1/2) scale in
// fp64, so the codes are those of the exact quotient.  (Dividing and comparing
// every element took twice as long.)  4099 positions of 8 heads of 128: 38 MB
// in 17 us, from cold caches.  What is left is one pass of loads, arithmetic,
// LDS and stores a block: 2080 blocks are about one round, and the
// chain of one block is what shows.
__device__ __forceinline__ void touched(const Kv4& c, int n, int n_touch, int& g, int& side, int& h, int& seq, int& pi) {
    int b = blockIdx.x;
    g = b % (c.hd / 64); b /= c.hd / 64;
    side = b & 1; b >>= 1;
    h = b % c.n_kv; b /= c.n_kv;
    pi = b % n_touch;
    seq = b / n_touch;
}
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4 c, const float* __restrict__ k,
                                                         const float* __restrict__ v, int n_new, int stride,
                                                         int n_touch, int vec) {
    __shared__ __align__(16) uint8_t code[kPage][68];    // values: a code a byte
    __shared__ __align__(16) uint8_t words[2048];        // keys: as they lie in the page
    const int hdg = c.hd / 64;
    int g, side, h, seq, pi;
    touched(c, n_new, n_touch, g, side, h, seq, pi);
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const int first = len - n_new;                       // position of row 0
    const int p = max(first, 0) / kPage + pi;
    if (bad) {
        if (threadIdx.x == 0) raise_table();
        return;
    }
    if (p * kPage >= len) return;
    const int tid = threadIdx.x, t = tid >> 2, cq = tid & 3;
    const int pos = p * kPage + t;
    const bool is_new = pos >= first && pos < len;
    const bool whole = p * kPage >= first && p * kPage + kPage <= len;
    float x[16];
    if (is_new) {
        const float* src = (side ? v : k) + ((size_t)seq * n_new + (pos - first)) * (size_t)stride + h * c.hd + 64 * g + 4 * cq;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (vec) {
                const float4 f = *(const float4*)(src + 16 * i);
                x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) x[4 * i + j] = src[16 * i + j];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = 0.f;
    }
    uint8_t* const pg = page_at(c, seq, p, h);
    if (!pg) {
        if (tid == 0) raise_table();
        return;
    }
    uint8_t* const part = pg + side * 36 * c.hd;
    // values: thread's two words of dim 32 j + 16 d1 + n, positions of quarter cv
    const int vd = 32 * (tid >> 7) + 16 * (tid & 1) + ((tid >> 1) & 15), cv = (tid >> 5) & 3;
    uint8_t* const vdst = part + (2 * g + (tid >> 7)) * 1024 + (cv * 16 + ((tid >> 1) & 15)) * 16 + (tid & 1) * 8;
    uint2 old = make_uint2(0u, 0u);
    if (side && !whole) old = *(const uint2*)vdst;       // what a page that is not all new keeps
    float lo = INFINITY, hi = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        nan |= x[i] != x[i];
        x[i] = __builtin_amdgcn_fmed3f(x[i], -65504.f, 65504.f);
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        lo = fminf(fminf(x[i], x[i + 1]), lo);
        hi = fmaxf(fmaxf(x[i], x[i + 1]), hi);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, o, kWave));
        hi = fmaxf(hi, __shfl_xor(hi, o, kWave));
        nan |= __shfl_xor((int)nan, o, kWave) != 0;
    }
    const uint32_t sb = nan ? 0x7e00u : f2h((hi - lo) / 15.0f);
    const float sc = h2f(sb);
    const uint32_t mb = nan ? 0x7e00u : f2h(lo + 8.0f * sc);
    const float mid = h2f(mb);
    if (is_new && cq == 0) ((uint32_t*)(part + 32 * c.hd))[g * 64 + slot_of(t)] = sb | (mb << 16);
    // a quotient held to -8 .. 7 plus 1.5 * 2^23 + 8 is rounded by the addition
    // (to nearest, ties to even) and has the code in its low byte
    constexpr float magic = 12582912.f + 8.f;
    const bool some = sc > 0.f;                          // codes 8 where the scale is 0 or NaN
    const float inv = some ? 1.0f / sc : 0.f, off = some ? mid : 0.f;
    uint32_t word[4];                                    // four codes, a byte each
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t cd[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float q = __builtin_amdgcn_fmed3f((x[4 * i + j] - off) * inv, -8.f, 7.f), r = q + magic;
            far = fmaxf(far, fabsf(q - (r - magic)));
            cd[j] = __builtin_bit_cast(uint32_t, r);
        }
        word[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(cd[3], cd[2], 0x0c0c0400), __builtin_amdgcn_perm(cd[1], cd[0], 0x0c0c0400), 0x05040100);
    }
    if (__any(some && far > 0.5f - 0x1p-17f)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            word[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float q = 0.f;
                if (sc > 0.f) {
                    q = fminf(fmaxf(rintf((x[4 * i + j] - mid) * inv), -8.f), 7.f);
                    const double d = (double)x[4 * i + j] - (double)mid;
                    const double up = (double)((q + 0.5f) * sc), dn = (double)((q - 0.5f) * sc);
                    const bool odd = ((int)q & 1) != 0;  // a tie goes to the even neighbour
                    if (q < 7.f && (d > up || (d == up && odd))) q += 1.f;
                    else if (q > -8.f && (d < dn || (d == dn && odd))) q -= 1.f;
                }
                word[i] |= (uint32_t)((int)q + 8) << (8 * j);
            }
        }
    }
    if (side == 0) {
        // dims 16 i + 4 cq ..: word cq / 2 of block i, half cq % 2
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t o = __shfl_xor(word[i], 1, kWave);
            const uint32_t w = word[i] | (o << 4);
            if (cq & 1) continue;
            if (whole) *(uint32_t*)(words + (t >> 5) * 1024 + (i * 16 + (t & 15)) * 16 + ((t >> 4) & 1) * 8 + (cq >> 1) * 4) = w;
            else if (is_new) *(uint32_t*)(part + key_off(t, g, i, hdg) + (cq >> 1) * 4) = w;
        }
        if (!whole) return;
        __syncthreads();
        if (tid < 128) *(uint4*)(part + ((tid >> 6) * hdg + g) * 1024 + (tid & 63) * 16) = *(const uint4*)(words + tid * 16);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) *(uint32_t*)&code[t][16 * i + 4 * cq] = word[i];
    __syncthreads();
    // a word of values holds eight positions of one dim: those that are not
    // new keep their nibbles (no other block writes these words)
    uint32_t w[2], m[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int r = 2 * cv + u;
        w[u] = m[u] = 0;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int hl = 0; hl < 2; hl++) {
                const int tt = 16 * i + 2 * r + hl, ps = p * kPage + tt;
                w[u] |= (uint32_t)code[tt][vd] << (8 * i + 4 * hl);
                if (ps >= first && ps < len) m[u] |= 0xfu << (8 * i + 4 * hl);
            }
    }
    if (m[0] | m[1]) *(uint2*)vdst = make_uint2((w[0] & m[0]) | (old.x & ~m[0]), (w[1] & m[1]) | (old.y & ~m[1]));
}

// ── read ─────────────────────────────────────────────────────────────────────
// The values of a sequence's last n positions: blocks and threads as above, a
// head's 64 dims of a page in LDS first.
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4 c, float* __restrict__ k, float* __restrict__ v, int n,
                                                       int stride, int n_touch, int vec) {
    __shared__ __align__(16) uint8_t words[2048];
    const int hdg = c.hd / 64;
    int g, side, h, seq, pi;
    touched(c, n, n_touch, g, side, h, seq, pi);
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const int first = len - n;
    const int p = max(first, 0) / kPage + pi;
    if (bad && threadIdx.x == 0) raise_table();
    if (p * kPage >= len) return;
    const uint8_t* const pg = page_at(c, seq, p, h);
    if (!pg && threadIdx.x == 0) raise_table();
    const int tid = threadIdx.x, t = tid >> 2, cq = tid & 3, pos = p * kPage + t;
    const uint8_t* const part = pg ? pg + side * 36 * c.hd : nullptr;
    uint32_t pr = 0x7e007e00u;
    if (pg && !bad) {
        if (tid < 128) {
            const int at = side ? (2 * g + (tid >> 6)) * 1024 : ((tid >> 6) * hdg + g) * 1024;
            *(uint4*)(words + tid * 16) = *(const uint4*)(part + at + (tid & 63) * 16);
        }
        pr = ((const uint32_t*)(part + 32 * c.hd))[g * 64 + slot_of(t)];
    }
    __syncthreads();
    if (pos < first || pos >= len) return;
    const float sc = h2f(pr), mid = h2f(pr >> 16);
    float* dst = (side ? v : k) + ((size_t)seq * n + (pos - first)) * (size_t)stride + h * c.hd + 64 * g + 4 * cq;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float y[4];
        if (side == 0) {
            const uint32_t w = *(const uint32_t*)(words + (t >> 5) * 1024 + (i * 16 + (t & 15)) * 16 + ((t >> 4) & 1) * 8 + (cq >> 1) * 4) >> (4 * (cq & 1));
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = (float)((int)(w >> (8 * j) & 15u) - 8);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int d = 16 * i + 4 * cq + j;
                y[j] = (float)((int)(words[val_off(d, (t & 15) >> 1) + (t >> 4)] >> (4 * (t & 1)) & 15) - 8);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = fmaf(sc, y[j], mid);
        if (vec) {
            *(float4*)(dst + 16 * i) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) dst[16 * i + j] = y[j];
        }
    }
}

// ── attention ────────────────────────────────────────────────────────────────
// The matrix cores multiply the codes as they lie.  The other operand of each
// product is written in four signed base-256 digits, x = step * (2^24 d0 + 2^16
// d1 + 2^8 d2 + d3), step a power of two that takes the largest element of a
// query, or of a page's p * scale, to 2^29 .. 2^30.  An element thus keeps its
// 24 bits down to 2^-6 of the largest, and 2^-30 of the largest below that;
// products and sums are exact in int32 and rounded where their digits are
// joined.  (With three digits, 22 bits, a query that has one channel of 3000
// among others of 1 left the output 4e-5 off.)  A tile is 4 query rows (a row
// is one head of one query) as the 16 rows of the MFMA's first operand: row
// 4 i + j is digit j of query row i.  The result leaves lane l with the digits'
// sums of query row l / 16 and column l % 16, so they are joined in the lane.
// Codes are 0 .. 15; a product with -8 in every place, used as the accumulator,
// centres them.
typedef int i4_t __attribute__((ext_vector_type(4)));
typedef int i4_alias __attribute__((ext_vector_type(4), may_alias));
typedef uint32_t u32_alias __attribute__((may_alias));

constexpr int kDigitBits = 30;                           // of the largest element: its highest digit is 64 or less
constexpr uint32_t kDigitOff = 0x00808080u;              // takes the low three digits to 0 .. 255
constexpr int kMaxSplit = 4096;                          // blocks of one row tile

__device__ __forceinline__ i4_t unpack16(uint32_t a, uint32_t b) {
    constexpr uint32_t M = 0x0f0f0f0fu;
    return i4_t{(int)(a & M), (int)((a >> 4) & M), (int)(b & M), (int)((b >> 4) & M)};
}
__device__ __forceinline__ i4_t mfma16(i4_t a, i4_t b, i4_t c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
// The upper and lower two digits' sums: 64 products of a pair with -8 .. 7 stay
// below 2^25, so each half is rounded by 2^-24 of itself at most.
__device__ __forceinline__ float upper_digits(i4_t c) { return (float)(c[0] * 256 + c[1]); }
__device__ __forceinline__ float lower_digits(i4_t c) { return (float)(c[2] * 256 + c[3]); }
__device__ __forceinline__ float join_digits(i4_t c) { return fmaf(upper_digits(c), 65536.f, lower_digits(c)); }
// A row's elements are multiplied by 2^digit_shift(their largest).
__device__ __forceinline__ int digit_shift(float most) { return kDigitBits - __builtin_amdgcn_frexp_expf(most); }
// v_exp_f32: at most one unit in the last place off, results below 2^-126 are 0
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// Largest value of the 16 lanes of a row, every lane getting it: v_max_f32
// with its first operand moved across lanes (the two wait states that a moved
// operand needs after its write stand before each).
__device__ __forceinline__ float row16_max(float v) {
    asm("s_nop 1\n\tv_max_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_ror:4 row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_ror:8 row_mask:0xf bank_mask:0xf\n\ts_nop 1" : "+v"(v));
    return v;
}
// Sum over the 16 lanes of a row, every lane getting it.
__device__ __forceinline__ float row16_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xF, 0xF, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xF, 0xF, false));
    return v;
}

// A lane's operands in a head's part of a page; at = 16 lane.  Pages that one
// block alone reads are loaded past the caches (NT): 604 MB are read at 7.0
// TB/s so, at 6.1 by ordinary loads.
template <bool NT>
__device__ __forceinline__ uint4 ld16(const uint8_t* p) {
    if constexpr (NT) return ld_stream16(p);
    else return *(const uint4*)p;
}
template <int HDG, bool NT>
__device__ __forceinline__ uint4 key_codes(const uint8_t* pg, int u, int g, unsigned at) {   // positions 32 u .., dims 64 g ..
    return ld16<NT>(pg + at + (u * HDG + g) * 1024);
}
template <int HDG, bool NT>
__device__ __forceinline__ uint4 key_pairs(const uint8_t* pg, int g, unsigned at) {          // positions 16 s + lane % 16
    return ld16<NT>(pg + (at & 255) + 2048 * HDG + g * 256);
}
template <int HDG, bool NT>
__device__ __forceinline__ uint4 val_codes(const uint8_t* pg, int j, unsigned at) {          // dims 32 j ..
    return ld16<NT>(pg + at + 2304 * HDG + j * 1024);
}
template <int HDG, bool NT>
__device__ __forceinline__ uint4 val_pairs(const uint8_t* pg, int g, unsigned at) {
    return ld16<NT>(pg + (at & 255) + 4352 * HDG + g * 256);
}
__device__ __forceinline__ uint32_t part4(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// What a launch of the attention kernels works on.
struct AttnArgs {
    float* out;
    const float* q;
    int n_heads, n_q, q_stride;
    float scale;                                         // log2(e) / sqrt(head_dim)
    int n_split, n_tile;                                 // most blocks of a row tile, row tiles of a KV head
    int chunk, quantum;                                  // pages of a block where a table row is full; a multiple of this
    uint32_t per_split;                                  // 2^32 / n_split, rounded up
    int tile_rows;                                       // query rows of a row tile
    float* part;                                         // [seq][KV head][row][split][head_dim], when n_split > 1
    float2* part_ml;                                     // [seq][KV head][row][split] maximum (log2) and sum
    float2* stat;                                        // [seq][KV head][row, stat_pad of them] row_stat(), when weights are wanted
    int stat_pad;
    i4_t* digits;                                        // [seq][KV head][4-row tile][group][lane]
    float* rowc;                                         // [seq][KV head][row][1 + groups] step * scale, sums of the query in steps
    float4* scores;                                      // [seq][KV head][page][tile][lane] scores (log2), -inf where not seen
};

// Pages of a block, for a sequence of `pages`: an equal share, whatever the
// table could hold (32 sequences of 4096 positions in tables of 32768: 32 us,
// 75 with blocks cut by the tables' size).
__host__ __device__ __forceinline__ int chunk_of(int pages, int n_split, uint32_t per_split, int quantum) {
    const uint32_t each = (uint32_t)(((uint64_t)(uint32_t)(pages + n_split - 1) * per_split) >> 32);
    return max((int)((each + quantum - 1) & ~(uint32_t)(quantum - 1)), quantum);
}
__device__ __forceinline__ int chunk_of(const AttnArgs& a, int len) {
    return a.n_split == 1 ? a.chunk : chunk_of((len + kPage - 1) / kPage, a.n_split, a.per_split, a.quantum);
}

// A row's maximum (log2) and the inverse of its sum, from which the weights
// are 2^(score - maximum) * inverse.  (Held as one number, maximum + log2(sum),
// the sum's share is rounded in steps of the maximum's: two tied scores of 2^25
// had weight 1 each, and a row at 10^4 weights that are all 3e-4 off.)  A row
// that sees nothing gives nothing: no score is above its maximum.
__device__ __forceinline__ float2 row_stat(float m, float sum) {
    return sum == 0.f ? make_float2(INFINITY, 0.f) : make_float2(m, 1.f / sum);
}

// Wavefronts a SIMD holds: what the registers of a page and RT tiles leave.
constexpr int attn_waves(int hdg, int rt) { return hdg * rt == 1 ? 4 : hdg * rt == 2 ? 3 : hdg * rt >= 8 && hdg > 2 ? 1 : 2; }

// Block: a share of the pages of one (sequence, KV head), RT tiles of 4 query
// rows, NW wavefronts that take the block's pages in turn, each with its own
// running maximum and sums, joined at the end.  4 sequences of 131071 positions,
// 8 KV heads of 128, 4 rows each: 604 MB in 96 us, 6.3 TB/s, of which HBM is the
// bound (7.0 by a kernel that only reads).  With 4096 positions it is the chain
// of a block: length, page number, codes, products, sums: 6 us.
template <int HDG, int RT, bool SCORES, int NW>
__global__ __launch_bounds__(64 * NW, attn_waves(HDG, RT)) void kv4_attn_kernel(Kv4 c, AttnArgs a) {
    constexpr int HD = 64 * HDG, ROWS = 4 * RT;
    __shared__ __align__(16) int8_t digs[RT * HDG * 1024];   // [tile][group][16][64]
    __shared__ __align__(16) int8_t turn[NW][HDG][4 * 320];   // a wavefront's p * scale digits, 64 B a row, a query row on 320
    __shared__ float rc[ROWS][1 + HDG];
    __shared__ float ob[NW][4][HD];
    __shared__ float mlw[NW][4][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lq = lane >> 4;
    // the KV head runs fastest over the blocks, so that blocks which share a
    // head's pages share an XCD's L2 where the heads are a multiple of 8; the
    // row tiles with the most positions come first
    int b = blockIdx.x;
    const int h = b % c.n_kv; b /= c.n_kv;
    const int rt = a.n_tile - 1 - b % a.n_tile; b /= a.n_tile;
    const int split = b % a.n_split, seq = b / a.n_split;
    const int grp = a.n_heads / c.n_kv, n_rows = a.n_q * grp;
    // the first page's number with the length, not behind it: that of a full row
    const int32_t* const ids = c.table + (size_t)seq * c.max_pages;
    int id0 = ld_uniform(ids + min(split * a.chunk + wave, c.max_pages - 1));
    bool bad;
    const int len = seq_len(c, seq, &bad), chunk = chunk_of(a, len);
    const int p0 = split * chunk;
    int p = p0 + wave;
    if (chunk != a.chunk) id0 = ld_uniform(ids + min(p, c.max_pages - 1));
    const int row0 = rt * ROWS;
    // the last position that each row sees; rows past the last copy it
    const int lim_min = len - a.n_q + row0 / grp, lim_max = len - a.n_q + min(row0 + ROWS - 1, n_rows - 1) / grp;
    const int pages = lim_max < 0 ? 0 : lim_max / kPage + 1;
    const int p1 = min(p0 + chunk, pages);
    if (split > 0 && p0 >= pages) return;
    int lim[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) lim[t] = len - a.n_q + min(row0 + 4 * t + lq, n_rows - 1) / grp;

    const size_t sh = (size_t)seq * c.n_kv + h;
    // a page no table entry names is left out of the sums (the block reports
    // it at its end and gives NaN): its wavefront goes on to its next page
    auto next_page = [&](int& p) -> const uint8_t* {
        for (; p < p1; p += NW) {
            const uint8_t* pg = page_of_wave(c, seq, p, h);
            if (pg) return pg;
            bad = true;
        }
        return nullptr;
    };
    uint4 kc[2][HDG], kp[HDG], vc[2 * HDG], vp[HDG];     // the page's codes and pairs
    unsigned at = 16 * lane;
    const uint8_t* pg = p < p1 ? page_by_id(c, id0, h) : nullptr;
    if (!pg && p < p1) {
        bad = true;
        p += NW;
        pg = next_page(p);
    }
    if (pg) {
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            kc[0][g] = key_codes<HDG, RT <= 2>(pg, 0, g, at);
            kc[1][g] = key_codes<HDG, RT <= 2>(pg, 1, g, at);
            kp[g] = key_pairs<HDG, RT <= 2>(pg, g, at);
        }
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            vc[2 * g] = val_codes<HDG, RT <= 2>(pg, 2 * g, at);
            vc[2 * g + 1] = val_codes<HDG, RT <= 2>(pg, 2 * g + 1, at);
            vp[g] = val_pairs<HDG, RT <= 2>(pg, g, at);
        }
    }

    // the query rows as digits
    for (int r = wave; r < ROWS; r += NW) {
        const int row = min(row0 + r, n_rows - 1);
        const float* src = a.q + ((size_t)seq * a.n_q + row / grp) * (size_t)a.q_stride + (h * grp + row % grp) * HD;
        float x[HDG], mx = 0.f;
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            x[g] = src[64 * g + lane];
            mx = fmaxf(mx, fabsf(x[g]));
        }
        mx = wave_max_dpp(mx);
        const bool inf = mx == INFINITY;                 // a row of NaN
        const int up = inf ? 0 : digit_shift(mx);
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            const uint32_t j = (inf ? 0u : (uint32_t)(int)rintf(ldexpf(x[g], up))) + kDigitOff;
            int8_t* d = digs + ((r >> 2) * HDG + g) * 1024 + (r & 3) * 256 + lane;
            d[0] = (int8_t)(j >> 24);
            d[64] = (int8_t)((j >> 16) ^ 0x80);
            d[128] = (int8_t)((j >> 8) ^ 0x80);
            d[192] = (int8_t)(j ^ 0x80);
            const float sum = ldexpf(wave_sum_dpp(x[g]), up);
            if (lane == 0) rc[r][1 + g] = inf ? NAN : sum;
        }
        if (lane == 0) rc[r][0] = ldexpf(a.scale, -up);
    }
    __syncthreads();
    i4_t qa[RT][HDG];
    float kf[RT], qsum[RT][HDG];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        kf[t] = rc[4 * t + lq][0];
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            qa[t][g] = *(const i4_alias*)(digs + (t * HDG + g) * 1024 + li * 64 + lq * 16);
            qsum[t][g] = rc[4 * t + lq][1 + g];
        }
    }
    if (a.digits && split == 0) {
        const size_t tiles = (n_rows + 3) / 4;
#pragma unroll
        for (int t = 0; t < RT; t++)
            if (t % NW == wave && row0 + 4 * t < n_rows) {
#pragma unroll
                for (int g = 0; g < HDG; g++) a.digits[((sh * tiles + row0 / 4 + t) * HDG + g) * 64 + lane] = qa[t][g];
                const int row = row0 + 4 * t + lq;
                if (li <= HDG && row < n_rows) a.rowc[(sh * n_rows + row) * (1 + HDG) + li] = rc[4 * t + lq][li];
            }
    }

    float m[RT], l[RT], o[RT][4 * HDG], om[RT][HDG];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < 4 * HDG; d++) o[t][d] = 0.f;
#pragma unroll
        for (int g = 0; g < HDG; g++) om[t][g] = 0.f;
    }
    const i4_t zero = {0, 0, 0, 0}, minus8 = {(int)0xf8f8f8f8, (int)0xf8f8f8f8, (int)0xf8f8f8f8, (int)0xf8f8f8f8};
    int8_t* const tw = &turn[wave][0][0];

    // One page, MASKED where some row of the block does not see all of it.
    // Each register is refilled from the wavefront's next page (nx) as soon as
    // its content has been taken apart; behind the last page every lane reads
    // one place of this page again (at = 0), which costs less than a branch.
    auto step = [&](int pos0, const uint8_t* nx, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        float e[RT][4], y[RT][4];                        // y: scores to keep
        {
            i4_t kb[4][HDG];
#pragma unroll
            for (int g = 0; g < HDG; g++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    kb[2 * u][g] = unpack16(kc[u][g].x, kc[u][g].y);
                    kb[2 * u + 1][g] = unpack16(kc[u][g].z, kc[u][g].w);
                }
#pragma unroll
            for (int g = 0; g < HDG; g++) {
                kc[0][g] = key_codes<HDG, RT <= 2>(nx, 0, g, at);
                kc[1][g] = key_codes<HDG, RT <= 2>(nx, 1, g, at);
            }
#pragma unroll
            for (int t = 0; t < RT; t++) {
                float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < HDG; g++) {
                    const i4_t init = mfma16(qa[t][g], minus8, zero);
#pragma unroll
                    for (int s = 0; s < 4; s++) {
                        const uint32_t pr = part4(kp[g], s);
                        const float f = join_digits(mfma16(qa[t][g], kb[s][g], init));
                        x[s] = fmaf(h2f(pr), f, fmaf(h2f(pr >> 16), qsum[t][g], x[s]));
                    }
                }
                // scores are rounded before the maximum is taken off: one fma
                // for both would leave the product's rounding in the
                // difference, which at scores of 2^31 is more than exp2 takes
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    x[s] *= kf[t];
                    if constexpr (MASKED) x[s] = pos0 + 16 * s + li <= lim[t] ? x[s] : -INFINITY;
                    if constexpr (SCORES) y[t][s] = x[s];
                }
                const float top = row16_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
                if (__any(top > m[t])) {
                    const float mn = fmaxf(m[t], top);
                    const float al = mn == -INFINITY ? 1.f : exp2_(m[t] - mn);
                    m[t] = mn;
                    l[t] *= al;
#pragma unroll
                    for (int d = 0; d < 4 * HDG; d++) o[t][d] *= al;
#pragma unroll
                    for (int g = 0; g < HDG; g++) om[t][g] *= al;
                }
                const float mk = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    e[t][s] = exp2_(x[s] - mk);
                    l[t] += e[t][s];
                }
            }
#pragma unroll
            for (int g = 0; g < HDG; g++) kp[g] = key_pairs<HDG, RT <= 2>(nx, g, at);
        }
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            i4_t vb[4];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                vb[2 * u] = unpack16(vc[2 * g + u].x, vc[2 * g + u].y);
                vb[2 * u + 1] = unpack16(vc[2 * g + u].z, vc[2 * g + u].w);
            }
            vc[2 * g] = val_codes<HDG, RT <= 2>(nx, 2 * g, at);
            vc[2 * g + 1] = val_codes<HDG, RT <= 2>(nx, 2 * g + 1, at);
#pragma unroll
            for (int t = 0; t < RT; t++) {
                float w[4];
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const uint32_t pr = part4(vp[g], s);
                    w[s] = e[t][s] * h2f(pr);
                    if constexpr (MASKED) {                  // stale pairs may be anything
                        const bool ok = pos0 + 16 * s + li <= lim[t];
                        w[s] = ok ? w[s] : 0.f;
                        om[t][g] += ok ? e[t][s] * h2f(pr >> 16) : 0.f;
                    } else {
                        om[t][g] = fmaf(e[t][s], h2f(pr >> 16), om[t][g]);
                    }
                }
                const float wm = row16_max(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])));
                const int up = digit_shift(wm);
                const float ws = ldexpf(1.f, -up), wu = ldexpf(1.f, 16 - up);
                uint32_t j[4];
#pragma unroll
                for (int s = 0; s < 4; s++) j[s] = (uint32_t)ldexpf(w[s], up) + kDigitOff;   // cut by 2^-30 of the largest
                // bytes of the four slots 4 li + s, one word a digit
                const uint32_t a01 = __builtin_amdgcn_perm(j[1], j[0], 0x05010400), a23 = __builtin_amdgcn_perm(j[3], j[2], 0x05010400);
                const uint32_t b01 = __builtin_amdgcn_perm(j[1], j[0], 0x07030602), b23 = __builtin_amdgcn_perm(j[3], j[2], 0x07030602);
                u32_alias* d = (u32_alias*)(tw + g * 1280 + lq * 320 + li * 4);
                d[0] = __builtin_amdgcn_perm(b23, b01, 0x07060302);
                d[16] = __builtin_amdgcn_perm(b23, b01, 0x05040100) ^ 0x80808080u;
                d[32] = __builtin_amdgcn_perm(a23, a01, 0x07060302) ^ 0x80808080u;
                d[48] = __builtin_amdgcn_perm(a23, a01, 0x05040100) ^ 0x80808080u;
                __builtin_amdgcn_wave_barrier();
                const i4_t wa = *(const i4_alias*)(tw + g * 1280 + (li >> 2) * 320 + (li & 3) * 64 + lq * 16);
                __builtin_amdgcn_wave_barrier();
                const i4_t init = mfma16(wa, minus8, zero);
#pragma unroll
                for (int d4 = 0; d4 < 4; d4++) {
                    const i4_t c = mfma16(wa, vb[d4], init);
                    o[t][4 * g + d4] = fmaf(upper_digits(c), wu, fmaf(lower_digits(c), ws, o[t][4 * g + d4]));
                }
            }
            vp[g] = val_pairs<HDG, RT <= 2>(nx, g, at);
        }
        if constexpr (SCORES) {
            // behind the next page's loads: a wait for a load waits for every store before it
#pragma unroll
            for (int t = 0; t < RT; t++) {
                typedef float f4_t __attribute__((ext_vector_type(4)));
                __builtin_nontemporal_store(f4_t{y[t][0], y[t][1], y[t][2], y[t][3]},
                                            (f4_t*)(a.scores + ((sh * c.max_pages + (pos0 >> 6)) * RT + t) * 64 + lane));
            }
        }
    };
    // pages that every row sees, then the others
    const int full = min(p1, (lim_min + 1) >> 6);
    auto run = [&](int end, auto masked) {
        while (pg && p < end) {
            int pn = p + NW;
            const uint8_t* nx = next_page(pn);
            if (!nx) at = 0;
            step(p * kPage, nx ? nx : pg, masked);
            pg = nx;
            p = pn;
        }
    };
    run(full, std::false_type{});
    run(p1, std::true_type{});

    // the wavefronts' sums, a tile at a time
    const bool any_bad = __syncthreads_or(bad);
    if (any_bad && tid == 0) raise_table();
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const float ls = row16_sum(l[t]);
        if (li == 0) {
            mlw[wave][lq][0] = m[t];
            mlw[wave][lq][1] = ls;
        }
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            const float mid = row16_sum(om[t][g]);
#pragma unroll
            for (int d = 0; d < 4; d++) ob[wave][lq][64 * g + 16 * d + li] = o[t][4 * g + d] + mid;
        }
        __syncthreads();
        const int r = wave, row = row0 + 4 * t + r;
        if (r < 4 && row < n_rows) {
            float mm = -INFINITY, f[NW], sum = 0.f;
#pragma unroll
            for (int w = 0; w < NW; w++) mm = fmaxf(mm, mlw[w][r][0]);
#pragma unroll
            for (int w = 0; w < NW; w++) {
                f[w] = mlw[w][r][0] == -INFINITY && mlw[w][r][1] == 0.f ? 0.f : exp2_(mlw[w][r][0] - mm);
                sum = fmaf(f[w], mlw[w][r][1], sum);
            }
            if (any_bad) sum = NAN;
            const size_t rr = sh * n_rows + row;
            const size_t to = a.n_split > 1 ? (rr * a.n_split + split) * HD
                                            : ((size_t)seq * a.n_q + row / grp) * (size_t)a.n_heads * HD + (h * grp + row % grp) * HD;
            float* dst = (a.n_split > 1 ? a.part : a.out) + to;
            const float norm = a.n_split > 1 ? 1.f : (sum == 0.f ? 0.f : 1.f / sum);
#pragma unroll
            for (int g = 0; g < HDG; g++) {
                float y = 0.f;
#pragma unroll
                for (int w = 0; w < NW; w++) y = fmaf(f[w], ob[w][r][64 * g + lane], y);
                dst[64 * g + lane] = y * norm;
            }
            if (lane == 0) {
                if (a.n_split > 1) a.part_ml[rr * a.n_split + split] = make_float2(mm, sum);
                else if (a.stat) a.stat[rr] = row_stat(mm, sum);
            }
        }
        __syncthreads();
    }
}

// ── attention of many rows ───────────────────────────────────────────────────
// From 33 query rows of a KV head on the sums are the f16 matrix cores': a row
// is one row of the MFMA, the query and p * scale are the sum of two fp16
// numbers, the codes are fp16 numbers -8 .. 7, and products are added in fp32.
// Such a sum has 22 bits, or steps of 2^-24 for numbers below 1/4: the query's
// largest element is taken to 2^14 .. 2^15, and p * scale by a factor of each
// row and 64 dims, so that the largest which the row has met there is at 2^7 or
// more, and what is lost is below 2^-32 of that, or 2^-85 of a p of 1.  (One
// factor for all rows, and a maximum that makes up for it, left rows 7e-5 off
// where values 2^24 times as large that they do not look at lie behind, or in
// other dims.)  That takes as many MFMAs as four digits in four rows, but no
// joining of digits, and the values' sums stay in the accumulators from page to
// page.  Block: 64 rows, 16 a wavefront; the four take a page's codes apart
// together, into LDS, as the matrix cores read them (a code word is a lane's 8
// elements of one MFMA: halves 0, 2, 4, 6, 1, 3, 5, 7 of its bytes' order).
//
// 512 queries of 32 heads on 8 KV heads of 128 over 4100 positions: 129 us, 32
// GFLOP at fp32's precision.  The vector ALU is what it waits for most, busy 62%
// of the time at the two wavefronts a SIMD that 228 registers leave: the
// exponentials, the rounding of 64 p * scale a row and group into halves, and two
// barriers a page.  (Three wavefronts a SIMD have 168 registers and spill; they
// serve 64 dims, with one register in scratch.  A running maximum by 16-lane
// reductions of every page's scores, as kv4_attn_kernel has it, took 10% longer;
// first factors that leave p * scale less room to grow, 2^11 .. 2^12 instead of
// 2^8 .. 2^9, are set again more often and took 3% longer.)
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_alias __attribute__((ext_vector_type(8), may_alias));
typedef float f4_t __attribute__((ext_vector_type(4)));
constexpr int kWideRows = 64;
constexpr float kTiny = 1e-30f;                          // a query below this counts as zero
constexpr float kNoMax = -0x1.fffffep127f;               // no score is lower
constexpr float kMostFactor = 0x1p60f;                   // times a p of 2^60 it is still a number

__device__ __forceinline__ f4_t mfma32(h8_t a, h8_t b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// A code word's eight numbers: 1024 + code as fp16 bits, less 1032.
__device__ __forceinline__ h8_t unpack_half(uint32_t w) {
    constexpr uint32_t M = 0x000f000fu, X = 0x64006400u;
    h8_t x;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t r = ((w >> (4 * i)) & M) | X;
        const h2_t y = __builtin_bit_cast(h2_t, r) + h2_t{(_Float16)-1032.f, (_Float16)-1032.f};
        x[2 * i] = y[0];
        x[2 * i + 1] = y[1];
    }
    return x;
}
// x - the low (HI: high) half of h
template <bool HI>
__device__ __forceinline__ float less_half(float x, uint32_t h) {
    float y;
    if constexpr (HI) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(y) : "v"(h), "v"(x));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(y) : "v"(h), "v"(x));
    return y;
}
// Two fp16 numbers, rounded to nearest: halves that are cut off are all too
// small, and the sum of the probabilities does not share that.
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2_t{a, b}, h2_t));
}

// Rows' constants for the weights, each array padded to whole blocks of rows.
struct WideRows {
    h8_t* q;                                             // [seq][KV head][16-row tile][group][2][high, low][lane]
    float *kf, *qsum;                                    // [..][row], [..][group][row]
    float2* stat;                                        // [..][row]
};
__device__ __forceinline__ int wide_pad(int n_rows) { return (n_rows + kWideRows - 1) / kWideRows * kWideRows; }

template <int HDG>
__global__ __launch_bounds__(256, HDG == 1 ? 3 : HDG == 2 ? 2 : 1) void kv4_attn_wide(Kv4 c, AttnArgs a, WideRows wr) {
    constexpr int HD = 64 * HDG, PR = 72;                // halves of a row of p * scale in LDS: 64 and 8 for the banks
    __shared__ __align__(16) uint8_t ops[16 * HDG * 1024];   // keys [position / 16][group][2], values [dim / 16][2]: a lane's 16 B
    __shared__ __align__(16) uint16_t pw[4][2][16 * PR];
    __shared__ __align__(16) uint32_t prs[2][HDG][64];   // the page's pairs, keys' then values'
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lq = lane >> 4;
    int b = blockIdx.x;
    const int h = b % c.n_kv; b /= c.n_kv;
    const int rt = a.n_tile - 1 - b % a.n_tile; b /= a.n_tile;
    const int split = b % a.n_split, seq = b / a.n_split;
    const int grp = a.n_heads / c.n_kv, n_rows = a.n_q * grp;
    const int32_t* const ids = c.table + (size_t)seq * c.max_pages;
    int id0 = ld_uniform(ids + min(split * a.chunk, c.max_pages - 1));
    bool bad;
    const int len = seq_len(c, seq, &bad), chunk = chunk_of(a, len);
    const int p0 = split * chunk;
    if (chunk != a.chunk) id0 = ld_uniform(ids + min(p0, c.max_pages - 1));
    const int base = len - a.n_q;                        // the first query's position
    const int lim_block = base + min(rt * kWideRows + kWideRows - 1, n_rows - 1) / grp;
    const int pages = lim_block < 0 ? 0 : lim_block / kPage + 1;
    const int p1 = min(p0 + chunk, pages);
    if (split > 0 && p0 >= pages) return;
    const int row0 = rt * kWideRows + wave * 16;
    const bool active = row0 < n_rows;
    const int lim_hi = base + min(row0 + 15, n_rows - 1) / grp;
    int lim[4];
#pragma unroll
    for (int r = 0; r < 4; r++) lim[r] = base + min(row0 + 4 * lq + r, n_rows - 1) / grp;
    const size_t sh = (size_t)seq * c.n_kv + h;

    // wavefronts 0, 1 take the keys apart (their halves u), 2, 3 the values
    const int chunk0 = wave < 2 ? wave * HDG * 1024 : 2304 * HDG + (wave - 2) * HDG * 1024;
    uint4 raw[HDG];
    uint32_t rawp[HDG];
    auto load = [&](const uint8_t* pg) {
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            raw[g] = *(const uint4*)(pg + chunk0 + g * 1024 + lane * 16);
            rawp[g] = *(const uint32_t*)(pg + (wave < 2 ? 2048 : 4352) * HDG + g * 256 + lane * 4);
        }
    };
    int p = p0;
    auto next_page = [&](int& p, int id) -> const uint8_t* {   // the same for every wavefront of the block
        while (p < p1) {
            const uint8_t* pg = page_by_id(c, id, h);
            if (pg) return pg;
            bad = true;
            if (++p < p1) id = ld_uniform(c.table + (size_t)seq * c.max_pages + p);
        }
        return nullptr;
    };
    const uint8_t* pg = next_page(p, id0);
    if (pg) load(pg);

    // the wavefront's rows: lane (li, lq) holds dims 16 lq .. + 15 of every 64
    h8_t qa[HDG][2][2];
    float kf[4], qsum[4][HDG];
    {
        const int row = min(row0 + li, n_rows - 1);
        const float* src = a.q + ((size_t)seq * a.n_q + row / grp) * (size_t)a.q_stride + (h * grp + row % grp) * HD + 16 * lq;
        float x[HDG][16], mx = 0.f;
#pragma unroll
        for (int g = 0; g < HDG; g++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                x[g][i] = src[64 * g + i];
                mx = fmaxf(mx, fabsf(x[g][i]));
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
        mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
        // a power of two takes the largest element to 2^14 .. 2^15
        const bool sane = mx > kTiny && mx < INFINITY;
        const int k = sane ? 15 - __builtin_amdgcn_frexp_expf(mx) : 0;
        float sum[HDG];
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            float t = 0.f;
#pragma unroll
            for (int kc = 0; kc < 2; kc++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int i = 8 * kc + (j < 4 ? 2 * j : 2 * j - 7);
                    const float y = mx > kTiny || mx != mx ? ldexpf(x[g][i], k) : x[g][i] * 0.f;
                    const _Float16 hi = (_Float16)y;
                    qa[g][kc][0][j] = hi;
                    qa[g][kc][1][j] = (_Float16)(y - (float)hi);
                    t += y;
                }
            t += __shfl_xor(t, 16, kWave);
            sum[g] = t + __shfl_xor(t, 32, kWave);
        }
        const float f = ldexpf(a.scale, -k);
#pragma unroll
        for (int r = 0; r < 4; r++) {                    // the rows of the results: 4 lq + r
            kf[r] = __shfl(f, 4 * lq + r, kWave);
#pragma unroll
            for (int g = 0; g < HDG; g++) qsum[r][g] = __shfl(sum[g], 4 * lq + r, kWave);
        }
        if (wr.q && split == 0) {
            const int pad = wide_pad(n_rows);
            h8_t* to = wr.q + (sh * (pad / 16) + row0 / 16) * HDG * 256 + lane;
#pragma unroll
            for (int g = 0; g < HDG; g++)
#pragma unroll
                for (int kc = 0; kc < 2; kc++)
#pragma unroll
                    for (int hl = 0; hl < 2; hl++) to[((g * 2 + kc) * 2 + hl) * 64] = qa[g][kc][hl];
            if (lq == 0) {
                wr.kf[sh * pad + row0 + li] = f;
#pragma unroll
                for (int g = 0; g < HDG; g++) wr.qsum[(sh * HDG + g) * pad + row0 + li] = sum[g];
                if (row0 + li >= n_rows) wr.stat[sh * pad + row0 + li] = row_stat(0.f, 0.f);
            }
        }
    }

    // p is 2^(score - m); the values' sums o are those of p * scale * f
    float m[4], l[4], om[4][HDG], f[4][HDG], fm[HDG];
    f4_t o[4 * HDG];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        m[r] = kNoMax;
        l[r] = 0.f;
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            om[r][g] = 0.f;
            f[r][g] = kMostFactor;
        }
    }
#pragma unroll
    for (int g = 0; g < HDG; g++) fm[g] = kMostFactor;
#pragma unroll
    for (int d = 0; d < 4 * HDG; d++) o[d] = f4_t{0.f, 0.f, 0.f, 0.f};
    uint16_t* const ph = pw[wave][0];
    uint16_t* const pl = pw[wave][1];

    auto step = [&](int pos0, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        float x[4][4];                                   // [row][position / 16]
#pragma unroll
        for (int s = 0; s < 4; s++) {
#pragma unroll
            for (int r = 0; r < 4; r++) x[r][s] = 0.f;
#pragma unroll
            for (int g = 0; g < HDG; g++) {
                f4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kc = 0; kc < 2; kc++) {
                    const h8_t kb = *(const h8_alias*)(ops + ((s * HDG + g) * 2 + kc) * 1024 + lane * 16);
                    d = mfma32(qa[g][kc][0], kb, d);
                    d = mfma32(qa[g][kc][1], kb, d);
                }
                const uint32_t pr = part4(*(const uint4*)&prs[0][g][4 * li], s);
#pragma unroll
                for (int r = 0; r < 4; r++) x[r][s] = fmaf(h2f(pr), d[r], fmaf(h2f(pr >> 16), qsum[r][g], x[r][s]));
            }
        }
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[r][s] *= kf[r];                        // rounded before m is taken off, as above
                if constexpr (MASKED) x[r][s] = pos0 + 16 * s + li <= lim[r] ? x[r][s] : -INFINITY;
            }
        float e[4][4];
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int s = 0; s < 4; s++) e[r][s] = exp2_(x[r][s] - m[r]);
        auto scale = [&](int g, int s) {
            const float v = h2f(part4(*(const uint4*)&prs[1][g][4 * li], s));
            return !MASKED || pos0 + 16 * s + li <= lim_hi ? v : 0.f;   // stale pairs may be anything
        };
        // m and f stay until a p is above 2^60 or a p * scale * f may not fit
        // fp16 (by the largest p and factor of the lane's four rows)
        float pm[4], high = 0.f, most = 0.f;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            pm[s] = fmaxf(fmaxf(e[0][s], e[1][s]), fmaxf(e[2][s], e[3][s]));
            high = fmaxf(high, pm[s]);
        }
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            float t = 0.f;
#pragma unroll
            for (int s = 0; s < 4; s++) t = fmaxf(t, pm[s] * scale(g, s));
            most = fmaxf(most, t * fm[g]);
        }
        if (__any(most > 65504.f || high > 0x1p60f)) {
            // m goes to the row's maximum.  A factor stays if the page's
            // largest p * scale is at 2^7 .. 65504 with it; else it makes up for
            // what p lost (rounded up: a maximum may creep), or takes that largest
            // to 2^8 .. 2^9.
#pragma unroll
            for (int g = 0; g < HDG; g++) fm[g] = 0.f;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float mn = fmaxf(m[r], row16_max(fmaxf(fmaxf(x[r][0], x[r][1]), fmaxf(x[r][2], x[r][3]))));
                const float al = exp2_(m[r] - mn), up = ldexpf(1.f, (int)ceilf(fminf(mn - m[r], 122.f)));
                m[r] = mn;
                l[r] *= al;
#pragma unroll
                for (int s = 0; s < 4; s++) e[r][s] = exp2_(x[r][s] - mn);
#pragma unroll
                for (int g = 0; g < HDG; g++) {
                    float t = 0.f;
#pragma unroll
                    for (int s = 0; s < 4; s++) t = fmaxf(t, e[r][s] * scale(g, s));
                    t = row16_max(t);
                    const float old = f[r][g], raised = fminf(old * up, kMostFactor);
                    float nf = raised;
                    if (old * t <= 65504.f && old * t >= 128.f) nf = old;
                    else if (raised * t > 65504.f) nf = ldexpf(1.f, 9 - __builtin_amdgcn_frexp_expf(t));
                    f[r][g] = nf;
                    fm[g] = fmaxf(fm[g], nf);
                    om[r][g] *= al;
                    const float of = ldexpf(al, __builtin_amdgcn_frexp_expf(nf) - __builtin_amdgcn_frexp_expf(old));
#pragma unroll
                    for (int d = 0; d < 4; d++) o[4 * g + d][r] *= of;
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int s = 0; s < 4; s++) l[r] += e[r][s];
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            float vs[4], vm[4];
#pragma unroll
            for (int s = 0; s < 4; s++) {
                vs[s] = scale(g, s);
                vm[s] = h2f(part4(*(const uint4*)&prs[1][g][4 * li], s) >> 16);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float w[4];
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    w[s] = e[r][s] * f[r][g] * vs[s];
                    if constexpr (MASKED) {              // a NaN that this row does not see
                        const bool ok = pos0 + 16 * s + li <= lim[r];
                        w[s] = ok ? w[s] : 0.f;
                        om[r][g] += ok ? e[r][s] * vm[s] : 0.f;
                    } else {
                        om[r][g] = fmaf(e[r][s], vm[s], om[r][g]);
                    }
                }
                // slots 4 li + s: quarter li / 4, half li / 2 % 2, then s = 0, 2 and s = 1, 3
                const uint32_t h02 = pack_half(w[0], w[2]), h13 = pack_half(w[1], w[3]);
                const uint32_t l02 = pack_half(less_half<false>(w[0], h02), less_half<true>(w[2], h02));
                const uint32_t l13 = pack_half(less_half<false>(w[1], h13), less_half<true>(w[3], h13));
                const int at = (4 * lq + r) * PR + (li >> 1) * 8 + (li & 1) * 2;
                *(u32_alias*)(ph + at) = h02;
                *(u32_alias*)(ph + at + 4) = h13;
                *(u32_alias*)(pl + at) = l02;
                *(u32_alias*)(pl + at + 4) = l13;
            }
            __builtin_amdgcn_wave_barrier();
            h8_t wa[2][2];
#pragma unroll
            for (int kc = 0; kc < 2; kc++) {
                wa[kc][0] = *(const h8_alias*)(ph + li * PR + lq * 16 + kc * 8);
                wa[kc][1] = *(const h8_alias*)(pl + li * PR + lq * 16 + kc * 8);
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int kc = 0; kc < 2; kc++) {
                h8_t vb[4];
#pragma unroll
                for (int d = 0; d < 4; d++) vb[d] = *(const h8_alias*)(ops + (8 * HDG + (4 * g + d) * 2 + kc) * 1024 + lane * 16);
#pragma unroll
                for (int hl = 0; hl < 2; hl++)
#pragma unroll
                    for (int d = 0; d < 4; d++) o[4 * g + d] = mfma32(wa[kc][hl], vb[d], o[4 * g + d]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // pages that every row of the block sees, then the others
    auto run = [&](int end, auto masked) {
      while (pg && p < end) {
        __syncthreads();                                 // the page before has been read
        {
            // chunk (u, g): operands (position / 16 = 2 u + i, g, half); value chunk j: (dim / 16 = 2 j + i, half)
#pragma unroll
            for (int g = 0; g < HDG; g++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int op = wave < 2 ? ((2 * wave + i) * HDG + g) * 2 : 8 * HDG + (2 * ((wave - 2) * HDG + g) + i) * 2;
                    *(h8_alias*)(ops + op * 1024 + lane * 16) = unpack_half(i ? raw[g].z : raw[g].x);
                    *(h8_alias*)(ops + (op + 1) * 1024 + lane * 16) = unpack_half(i ? raw[g].w : raw[g].y);
                }
            if (!(wave & 1)) {
#pragma unroll
                for (int g = 0; g < HDG; g++) prs[wave >> 1][g][lane] = rawp[g];
            }
        }
        int pn = p + 1;
        const uint8_t* nx = pn < p1 ? next_page(pn, ld_uniform(c.table + (size_t)seq * c.max_pages + pn)) : nullptr;
        if (nx) load(nx);
        __syncthreads();
        if (active && p * kPage <= lim_hi) step(p * kPage, masked);
        pg = nx;
        p = pn;
      }
    };
    run(min(p1, (base + rt * kWideRows / grp + 1) >> 6), std::false_type{});
    run(p1, std::true_type{});

    if (bad && tid == 0) raise_table();
    if (!active) return;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int row = row0 + 4 * lq + r;
        float sum = row16_sum(l[r]);
        if (bad) sum = NAN;
        const size_t rr = sh * n_rows + row;
        const bool in = row < n_rows;
        float* dst = a.n_split > 1 ? a.part + (rr * a.n_split + split) * HD
                                   : a.out + ((size_t)seq * a.n_q + row / grp) * (size_t)a.n_heads * HD + (h * grp + row % grp) * HD;
        const float norm = a.n_split > 1 ? (bad ? NAN : 1.f) : (sum == 0.f ? 0.f : 1.f / sum);
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            const float mid = row16_sum(om[r][g]), back = 1.f / f[r][g];
#pragma unroll
            for (int d = 0; d < 4; d++)
                if (in) dst[64 * g + 16 * d + li] = fmaf(o[4 * g + d][r], back, mid) * norm;
        }
        if (in && li == 0) {
            if (a.n_split > 1) a.part_ml[rr * a.n_split + split] = make_float2(m[r], sum);
            else if (wr.stat) wr.stat[sh * wide_pad(n_rows) + row] = row_stat(m[r], sum);
        }
    }
}

// Accumulated weights of many rows: block (KV head, page, sequence); every
// wavefront holds the page's keys and takes 16-row tiles in turn.  2048 rows
// of 8 KV heads of 128 over 4100 positions: 55 us, in which every page reads
// all rows' halves from L2, 8 KB a tile, 10 TB/s.
template <int HDG, int NW>
__global__ __launch_bounds__(64 * NW) void kv4_weights_wide(Kv4 c, AttnArgs a, WideRows wr, const float* win, float* wout) {
    __shared__ float part[NW][kPage];
    const int lane = threadIdx.x & 63, li = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int b = blockIdx.x;
    const int h = b % c.n_kv; b /= c.n_kv;
    const int p = b % c.max_pages, seq = b / c.max_pages;
    const int grp = a.n_heads / c.n_kv, n_rows = a.n_q * grp, pad = wide_pad(n_rows), tiles = (n_rows + 15) / 16;
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const size_t sh = (size_t)seq * c.n_kv + h;
    const size_t at = (sh * c.max_pages + p) * kPage + lane;
    if (p * kPage >= len) {
        if (wave == 0) wout[at] = 0.f;
        return;
    }
    const uint8_t* pg = page_of_wave(c, seq, p, h);
    if (pg && !bad) {
        h8_t kb[4][HDG][2];
        uint4 kp[HDG];
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            kp[g] = key_pairs<HDG, false>(pg, g, 16 * lane);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint4 x = key_codes<HDG, false>(pg, u, g, 16 * lane);
                kb[2 * u][g][0] = unpack_half(x.x);
                kb[2 * u][g][1] = unpack_half(x.y);
                kb[2 * u + 1][g][0] = unpack_half(x.z);
                kb[2 * u + 1][g][1] = unpack_half(x.w);
            }
        }
        // queries before the page's first position see nothing of it
        const int base = len - a.n_q, t0 = max(0, p * kPage - base) * grp / 16;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int t = t0 + wave; t < tiles; t += NW) {
            const h8_t* q = wr.q + (sh * (pad / 16) + t) * HDG * 256 + lane;
            const int row = 16 * t + 4 * lq;
            const f4_t kf = *(const f4_t*)(wr.kf + sh * pad + row);
            float2 st[4];
#pragma unroll
            for (int r = 0; r < 4; r++) st[r] = wr.stat[sh * pad + row + r];
            float x[4][4];
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int s = 0; s < 4; s++) x[r][s] = 0.f;
#pragma unroll
            for (int g = 0; g < HDG; g++) {
                const f4_t qs = *(const f4_t*)(wr.qsum + (sh * HDG + g) * pad + row);
                h8_t qa[2][2];
#pragma unroll
                for (int kc = 0; kc < 2; kc++)
#pragma unroll
                    for (int hl = 0; hl < 2; hl++) qa[kc][hl] = q[((g * 2 + kc) * 2 + hl) * 64];
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    f4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kc = 0; kc < 2; kc++) {
                        d = mfma32(qa[kc][0], kb[s][g][kc], d);
                        d = mfma32(qa[kc][1], kb[s][g][kc], d);
                    }
                    const uint32_t pr = part4(kp[g], s);
#pragma unroll
                    for (int r = 0; r < 4; r++) x[r][s] = fmaf(h2f(pr), d[r], fmaf(h2f(pr >> 16), qs[r], x[r][s]));
                }
            }
            if (p * kPage + kPage - 1 <= base + 16 * t / grp) {
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int s = 0; s < 4; s++) acc[s] = fmaf(exp2_(x[r][s] * kf[r] - st[r].x), st[r].y, acc[s]);
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int lim = base + min(row + r, n_rows - 1) / grp;
#pragma unroll
                    for (int s = 0; s < 4; s++)
                        acc[s] += p * kPage + 16 * s + li <= lim ? exp2_(x[r][s] * kf[r] - st[r].x) * st[r].y : 0.f;
                }
            }
        }
#pragma unroll
        for (int s = 0; s < 4; s++) {
            acc[s] += __shfl_xor(acc[s], 16, kWave);
            acc[s] += __shfl_xor(acc[s], 32, kWave);
        }
        part[wave][lane] = lq == 0 ? acc[0] : lq == 1 ? acc[1] : lq == 2 ? acc[2] : acc[3];
    } else {
        if (threadIdx.x == 0) raise_table();
        part[wave][lane] = NAN;
    }
    __syncthreads();
    if (wave) return;
    float add = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w++) add += part[w][lane];
    wout[at] = p * kPage + lane < len ? win[at] + add : 0.f;
}

// Blocks of a row's tile that had work: as kv4_attn_kernel cut the pages.
__device__ __forceinline__ int splits_of(const AttnArgs& a, int len, int row, int grp, int n_rows) {
    const int last = min(row / a.tile_rows * a.tile_rows + a.tile_rows, n_rows) - 1;
    const int lim = len - a.n_q + last / grp;
    const int chunk = chunk_of(a, len);
    return lim < 0 ? 1 : (lim / kPage + chunk) / chunk;
}

// A page's keys, and the probabilities of its positions summed over the rows of
// tiles t0, t0 + dt, .. < t1: lane l of sum() returns position l's (the rows'
// digits, step * scale, sums, row_stat() and last positions as the callers give
// them).
template <int HDG>
struct PageWeights {
    uint4 kc[2][HDG], kp[HDG];
    __device__ __forceinline__ void load(const uint8_t* pg, int lane) {
        const unsigned at = 16 * lane;
#pragma unroll
        for (int g = 0; g < HDG; g++) {
            kc[0][g] = key_codes<HDG, false>(pg, 0, g, at);
            kc[1][g] = key_codes<HDG, false>(pg, 1, g, at);
            kp[g] = key_pairs<HDG, false>(pg, g, at);
        }
    }
    template <class Rows>
    __device__ __forceinline__ float sum(const i4_t* digits, int pos0, int lane, int t0, int t1, int dt, Rows rows) const {
        const int li = lane & 15, lq = lane >> 4;
        const i4_t zero = {0, 0, 0, 0}, minus8 = {(int)0xf8f8f8f8, (int)0xf8f8f8f8, (int)0xf8f8f8f8, (int)0xf8f8f8f8};
        i4_t kb[4][HDG], qa[HDG];
#pragma unroll
        for (int g = 0; g < HDG; g++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                kb[2 * u][g] = unpack16(kc[u][g].x, kc[u][g].y);
                kb[2 * u + 1][g] = unpack16(kc[u][g].z, kc[u][g].w);
            }
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        float kf, qs[HDG];
        float2 st;
        int lim;                                         // the last position that the lane's row sees
        if (t0 < t1) {
#pragma unroll
            for (int g = 0; g < HDG; g++) qa[g] = digits[((size_t)t0 * HDG + g) * 64 + lane];
            rows(t0, lq, kf, st, qs, lim);
        }
        for (int t = t0; t < t1; t += dt) {
            // the next tile's rows are loaded while this one's are multiplied
            i4_t qn[HDG];
            float kfn = 0.f, qsn[HDG];
            float2 stn = make_float2(0.f, 0.f);
            int limn = -1;
#pragma unroll
            for (int g = 0; g < HDG; g++) {
                qn[g] = zero;
                qsn[g] = 0.f;
            }
            if (t + dt < t1) {
#pragma unroll
                for (int g = 0; g < HDG; g++) qn[g] = digits[((size_t)(t + dt) * HDG + g) * 64 + lane];
                rows(t + dt, lq, kfn, stn, qsn, limn);
            }
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < HDG; g++) {
                const i4_t init = mfma16(qa[g], minus8, zero);
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const uint32_t pr = part4(kp[g], s);
                    x[s] = fmaf(h2f(pr), join_digits(mfma16(qa[g], kb[s][g], init)), fmaf(h2f(pr >> 16), qs[g], x[s]));
                }
            }
#pragma unroll
            for (int s = 0; s < 4; s++) acc[s] += pos0 + 16 * s + li <= lim ? exp2_(x[s] * kf - st.x) * st.y : 0.f;
            kf = kfn;
            st = stn;
            lim = limn;
#pragma unroll
            for (int g = 0; g < HDG; g++) {
                qa[g] = qn[g];
                qs[g] = qsn[g];
            }
        }
#pragma unroll
        for (int s = 0; s < 4; s++) {
            acc[s] += __shfl_xor(acc[s], 16, kWave);
            acc[s] += __shfl_xor(acc[s], 32, kWave);
        }
        return lq == 0 ? acc[0] : lq == 1 ? acc[1] : lq == 2 ? acc[2] : acc[3];
    }
};

// Joins up to 8 splits of many rows: a wavefront a row, where kv4_attn_finish has
// a block a row.  Whole calls by the one and the other: 16384 rows of 128 dims
// 131 and 150 us with 2 splits, 129 and 143 with 8, 148 and 161 with 16; 2560
// rows 40 and 41 with 8, 57 and 55 with 24; 320 rows 28 and 27 with 8, 24 and 20
// with 16.
constexpr int kFewSplits = 8;
template <int HDG>
__global__ __launch_bounds__(256) void kv4_attn_join(Kv4 c, AttnArgs a, size_t rows) {
    constexpr int HD = 64 * HDG;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = a.n_heads / c.n_kv, n_rows = a.n_q * grp;
    const size_t rr = (size_t)blockIdx.x * 4 + wave;
    if (rr >= rows) return;
    const size_t sh = rr / n_rows;
    const int row = rr % n_rows, h = sh % c.n_kv, seq = sh / c.n_kv;
    bool bad;
    const int n = splits_of(a, seq_len(c, seq, &bad), row, grp, n_rows);
    const float2* ml = a.part_ml + rr * a.n_split;
    const float* po = a.part + rr * a.n_split * HD + lane;
    float mm = -INFINITY, sum = 0.f, y[HDG] = {};
    for (int i = 0; i < n; i++) {
        const float2 v = ml[i];
        const float mn = fmaxf(mm, v.x);
        const float f0 = mm == -INFINITY && sum == 0.f ? 0.f : exp2_(mm - mn), f1 = v.x == -INFINITY && v.y == 0.f ? 0.f : exp2_(v.x - mn);
        mm = mn;
        sum = fmaf(f1, v.y, sum * f0);
#pragma unroll
        for (int g = 0; g < HDG; g++) y[g] = fmaf(f1, po[(size_t)i * HD + 64 * g], y[g] * f0);
    }
    float* dst = a.out + ((size_t)seq * a.n_q + row / grp) * (size_t)a.n_heads * HD + (h * grp + row % grp) * HD + lane;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int g = 0; g < HDG; g++) dst[64 * g] = y[g] * inv;
    if (lane == 0 && a.stat) a.stat[sh * a.stat_pad + row] = row_stat(mm, sum);
}

// A query row's row_stat() from its splits, by the 16 lanes of a row.
__device__ __forceinline__ float2 joined_stat(const float2* ml, int n, int li) {
    float m = -INFINITY, s = 0.f;
    for (int i = li; i < n; i += 16) m = fmaxf(m, ml[i].x);
    m = row16_max(m);
    for (int i = li; i < n; i += 16) {
        const float2 v = ml[i];
        s = fmaf(v.x == -INFINITY && v.y == 0.f ? 0.f : exp2_(v.x - m), v.y, s);
    }
    return row_stat(m, row16_sum(s));
}

// What is left after the pages' blocks.  Blocks below n_join join the splits
// of a query row: 16 HDG threads hold four dims each, the other threads take
// other splits, so that all partial sums are in flight together.  The others,
// where one row tile holds all rows, take a page a wavefront and turn the
// scores that the first kernel kept into weights; they take row_stat()
// from the splits' maxima and sums themselves, so that they need not wait for the
// joining blocks.  At 32 sequences of up to 4096 positions, 8 KV heads of 128,
// this launch takes 10 us, and keeping the scores costs the first 1.2 us, by
// nontemporal stores behind a page's loads (9 us by ordinary ones, which the
// next loads wait for).  Scoring the pages again in a launch of their own takes
// the call from 44 to 48 us where all are full, in tables of 32768 positions from
// 66 to 68.
template <int HDG, int RT>
__global__ __launch_bounds__(256) void kv4_attn_finish(Kv4 c, AttnArgs a, unsigned n_join, const float* win, float* wout) {
    constexpr int HD = 64 * HDG, TD = HD / 4, CLS = 256 / TD;
    __shared__ float f[kMaxSplit];
    __shared__ float4 ob[CLS][TD];
    __shared__ float red[2][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = a.n_heads / c.n_kv, n_rows = a.n_q * grp;
    bool bad;
    if (blockIdx.x < n_join) {
        const size_t rr = blockIdx.x, sh = rr / n_rows;
        const int row = rr % n_rows, h = sh % c.n_kv, seq = sh / c.n_kv;
        const int len = seq_len(c, seq, &bad);
        const int n = splits_of(a, len, row, grp, n_rows);
        const float2* ml = a.part_ml + rr * a.n_split;
        const int td = tid % TD, cl = tid / TD;
        const float4* po = (const float4*)(a.part + rr * a.n_split * HD) + td;
        float4 first = make_float4(0.f, 0.f, 0.f, 0.f);
        if (cl < CLS && cl < n) first = po[(size_t)cl * TD];
        float mm = -INFINITY;
        for (int i = tid; i < n; i += 256) mm = fmaxf(mm, ml[i].x);
        mm = wave_max_dpp(mm);
        if (lane == 0) red[0][wave] = mm;
        __syncthreads();
        mm = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        float sum = 0.f;
        for (int i = tid; i < n; i += 256) {
            const float2 v = ml[i];
            const float w = v.x == -INFINITY && v.y == 0.f ? 0.f : exp2_(v.x - mm);
            f[i] = w;
            sum = fmaf(w, v.y, sum);
        }
        sum = wave_sum_dpp(sum);
        if (lane == 0) red[1][wave] = sum;
        __syncthreads();
        sum = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
        if (cl < CLS) {
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            if (cl < n) {
                const float w = f[cl];
                y = make_float4(w * first.x, w * first.y, w * first.z, w * first.w);
            }
#pragma unroll 4
            for (int i = cl + CLS; i < n; i += CLS) {
                const float4 v = po[(size_t)i * TD];
                const float w = f[i];
                y.x = fmaf(w, v.x, y.x);
                y.y = fmaf(w, v.y, y.y);
                y.z = fmaf(w, v.z, y.z);
                y.w = fmaf(w, v.w, y.w);
            }
            ob[cl][td] = y;
        }
        __syncthreads();
        if (tid < HD) {
            float y = 0.f;
#pragma unroll
            for (int k = 0; k < CLS; k++) y += ((const float*)&ob[k][0])[tid];
            a.out[((size_t)seq * a.n_q + row / grp) * (size_t)a.n_heads * HD + (h * grp + row % grp) * HD + tid] =
                sum == 0.f ? 0.f : y / sum;
        }
        if (tid == 0 && a.stat) a.stat[sh * a.stat_pad + row] = row_stat(mm, sum);
        return;
    }
    unsigned b = blockIdx.x - n_join;
    const int h = b % c.n_kv; b /= c.n_kv;
    const int np = (c.max_pages + 3) / 4;
    const int p = b % np * 4 + wave, seq = b / np;
    if (p >= c.max_pages) return;
    const size_t sh = (size_t)seq * c.n_kv + h;
    const int len = seq_len(c, seq, &bad);
    const size_t at = (sh * c.max_pages + p) * kPage + lane;
    if (p * kPage >= len) {
        wout[at] = 0.f;
        return;
    }
    const float old = win[at];
    float4 x[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) x[t] = a.scores[((sh * c.max_pages + p) * RT + t) * 64 + lane];
    const int n = splits_of(a, len, 0, grp, n_rows);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int lq = lane >> 4;
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const int r = 4 * t + lq;
        float2 st = joined_stat(a.part_ml + (sh * n_rows + min(r, n_rows - 1)) * a.n_split, n, lane & 15);
        if (r >= n_rows) st = row_stat(0.f, 0.f);
        acc[0] = fmaf(exp2_(x[t].x - st.x), st.y, acc[0]);
        acc[1] = fmaf(exp2_(x[t].y - st.x), st.y, acc[1]);
        acc[2] = fmaf(exp2_(x[t].z - st.x), st.y, acc[2]);
        acc[3] = fmaf(exp2_(x[t].w - st.x), st.y, acc[3]);
    }
#pragma unroll
    for (int s = 0; s < 4; s++) {
        acc[s] += __shfl_xor(acc[s], 16, kWave);
        acc[s] += __shfl_xor(acc[s], 32, kWave);
    }
    const float add = lq == 0 ? acc[0] : lq == 1 ? acc[1] : lq == 2 ? acc[2] : acc[3];
    wout[at] = p * kPage + lane < len ? old + add : 0.f;
}

// Accumulated weights where the rows fill several tiles: block (KV head, page,
// sequence), its wavefronts take the tiles in turn.
template <int HDG, int NW>
__global__ __launch_bounds__(64 * NW) void kv4_attn_weights(Kv4 c, AttnArgs a, const float* win, float* wout) {
    __shared__ float part[NW][kPage];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int b = blockIdx.x;
    const int h = b % c.n_kv; b /= c.n_kv;
    const int p = b % c.max_pages, seq = b / c.max_pages;
    const int grp = a.n_heads / c.n_kv, n_rows = a.n_q * grp, tiles = (n_rows + 3) / 4;
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const size_t sh = (size_t)seq * c.n_kv + h;
    const size_t at = (sh * c.max_pages + p) * kPage + lane;
    if (p * kPage >= len) {
        if (wave == 0) wout[at] = 0.f;
        return;
    }
    const uint8_t* pg = page_of_wave(c, seq, p, h);
    if (pg && !bad) {
        PageWeights<HDG> pw;
        pw.load(pg, lane);
        // queries before the page's first position see nothing of it
        const int t0 = max(0, p * kPage - (len - a.n_q)) * grp / 4;
        part[wave][lane] = pw.sum(a.digits + sh * tiles * HDG * 64, p * kPage, lane, t0 + wave, tiles, NW,
            [&](int t, int lq, float& kf, float2& st, float* qs, int& lim) {
                const int r = 4 * t + lq, row = min(r, n_rows - 1);
                const float* rcp = a.rowc + (sh * n_rows + row) * (1 + HDG);
                kf = rcp[0];
                st = a.stat[sh * n_rows + row];
#pragma unroll
                for (int g = 0; g < HDG; g++) qs[g] = rcp[1 + g];
                lim = r < n_rows ? len - a.n_q + row / grp : -1;
            });
    } else {
        if (threadIdx.x == 0) raise_table();
        part[wave][lane] = NAN;
    }
    __syncthreads();
    if (wave) return;
    float add = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w++) add += part[w][lane];
    wout[at] = p * kPage + lane < len ? win[at] + add : 0.f;
}

// ── eviction ─────────────────────────────────────────────────────────────────
// Order-preserving integer of a weight: NaN lowest, -0 and +0 alike.
__device__ __forceinline__ uint32_t rank_of(float w) {
    if (w != w) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kSelMost = kSelThreads * 16;               // longest row of the one-block selection: 16 ranks a thread

constexpr int kBins = 2048;
__device__ __forceinline__ int bin_shift(int level) { return level == 0 ? 21 : level == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t bin_of(uint32_t rank, int level) {
    return (rank >> bin_shift(level)) & (level == 2 ? 1023u : 2047u);
}

// The bin that holds the need-th largest: thread t brings the counts of bins
// hi = 2046 - 2 t (lo) and hi + 1 (up).  Returns the bin and takes what lies
// above it off `need`.  Two barriers before the result is read, none after.
struct BinPick {
    uint32_t scan[kSelWaves];
    uint32_t found[2];
};
__device__ __forceinline__ uint32_t pick_bin(BinPick& sh, uint32_t lo, uint32_t up, uint32_t& need) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = kBins - 2 * (tid + 1);
    uint32_t run = lo + up;                              // counts of this thread's bins and all higher ones
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(run, o, kWave);
        if (lane >= o) run += v;
    }
    if (lane == 63) sh.scan[wave] = run;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSelWaves; k++) run += k < wave ? sh.scan[k] : 0u;
    const uint32_t higher = run - (lo + up);
    if (higher < need && run >= need) {                  // one thread
        const bool top = higher + up >= need;
        sh.found[0] = top ? hi + 1 : hi;
        sh.found[1] = top ? higher : higher + up;
    }
    __syncthreads();
    need -= sh.found[1];
    return sh.found[0];
}

// Rows of up to 16384 positions: block (KV head, sequence), the ranks in
// registers.  Their top 11, middle 11 and low 10 bits in turn are counted in
// LDS among the ranks that share the bits found before, which gives the
// need-th largest rank and how many of those equal to it are kept.  (Bit by
// bit with ballots and a barrier a bit took 21 us at 4096 positions.)
template <int KEYS>
__global__ __launch_bounds__(kSelThreads) void kv4_select(Kv4 c, const float* __restrict__ w, int budget, int sink,
                                                          int recent, int32_t* __restrict__ kept) {
    __shared__ __align__(16) uint32_t hist[3][kBins];
    __shared__ BinPick bp;
    __shared__ int cnt2[kSelWaves][2];
    const int seq = blockIdx.x / c.n_kv;
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const float* wr = w + (size_t)blockIdx.x * c.max_pages * kPage;
    int32_t* kr = kept + (size_t)blockIdx.x * budget;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (bad && tid == 0) raise_table();
    if (bad || len <= budget) {
        for (int i = tid; i < budget; i += kSelThreads) kr[i] = !bad && i < len ? i : -1;
        return;
    }
    const int z = len - recent;                          // candidates [sink, z)
    const int need = budget - sink - recent;
    const int per = (len + kSelWaves * 64 - 1) / (kSelWaves * 64) * 64;   // positions of a wavefront
    const int a = wave * per, e = min(len, a + per);
    uint32_t key[KEYS];
#pragma unroll
    for (int j = 0; j < KEYS; j++) {
        const int i = a + 64 * j + lane;
        key[j] = i < e && i >= sink && i < z ? rank_of(wr[i]) : 0u;
    }
    for (int i = tid; i < 3 * kBins / 4; i += kSelThreads) ((uint4*)&hist[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    uint32_t cut = 0, left = need;
    const bool choose = need > 0;
    if (choose)
#pragma unroll
        for (int lv = 0; lv < 3; lv++) {
            const uint32_t known = lv == 0 ? 0u : lv == 1 ? ~0u << 21 : ~0u << 10;
#pragma unroll
            for (int j = 0; j < KEYS; j++) {
                const int i = a + 64 * j + lane;
                if (64 * j < per && i < e && i >= sink && i < z && (key[j] & known) == cut)
                    atomicAdd(&hist[lv][bin_of(key[j], lv)], 1u);
            }
            __syncthreads();
            const uint2 v = *(const uint2*)&hist[lv][kBins - 2 * (tid + 1)];
            cut |= pick_bin(bp, v.x, v.y, left) << bin_shift(lv);
        }
    int above = 0, equal = 0;
#pragma unroll
    for (int j = 0; j < KEYS; j++)
        if (64 * j < per) {
            const int i = a + 64 * j + lane;
            const bool in = i < e, cand = in && i >= sink && i < z;
            above += __popcll(__ballot(in && (!cand || (choose && key[j] > cut))));
            equal += __popcll(__ballot(cand && choose && key[j] == cut));
        }
    if (lane == 0) { cnt2[wave][0] = above; cnt2[wave][1] = equal; }
    __syncthreads();
    int total = 0, at = 0, eqs = 0;                      // all that are sure; kept and equal before this stretch
#pragma unroll
    for (int k = 0; k < kSelWaves; k++) {
        total += cnt2[k][0];
        if (k < wave) {
            at += cnt2[k][0];
            eqs += cnt2[k][1];
        }
    }
    const int equals = budget - total;                   // how many of the equal ones are kept
    at += min(eqs, equals);
    const unsigned long long low = (1ull << lane) - 1;
#pragma unroll
    for (int j = 0; j < KEYS; j++)
        if (64 * j < per) {
            const int i = a + 64 * j + lane;
            const bool in = i < e, cand = in && i >= sink && i < z, eq = cand && choose && key[j] == cut;
            const unsigned long long be = __ballot(eq);
            const bool keep = in && (!cand || (choose && key[j] > cut) || (eq && eqs + __popcll(be & low) < equals));
            const unsigned long long bk = __ballot(keep);
            if (keep) kr[at + __popcll(bk & low)] = i;
            at += __popcll(bk);
            eqs += __popcll(be);
        }
}

// Longer rows: up to 32 blocks a row, each with its own segment, in four
// launches.  Launches 0, 1, 2 count a segment's ranks by their top 11, middle
// 11 and low 10 bits, among those that share the bits found before; every
// block of the next launch adds up the segments' counts and so finds the next
// bits for itself.  Launch 3 takes what the segments before its own keep from
// the same counts, and emits.
constexpr int kSegs = 32;
struct LongSel {
    uint32_t* hist;                                      // [row][launch 0, 1, 2][segment][kBins]
    uint32_t* above;                                     // [row][launch 1, 2][segment] ranks that the bits found last put above the cut
    uint32_t* state;                                     // [row][launch 1, 2][2] cut and need behind that launch
    int seg, n_seg;                                      // positions of a segment, segments of a row
    int budget, sink, recent;
};

template <int LEVEL>
__global__ __launch_bounds__(kSelThreads) void kv4_select_long(Kv4 c, LongSel q, const float* __restrict__ w,
                                                               int32_t* __restrict__ kept) {
    __shared__ __align__(16) uint32_t hist[LEVEL < 3 ? kBins : 4];
    __shared__ BinPick bp;
    __shared__ int cnt2[kSelWaves][3];
    const int row = blockIdx.x / q.n_seg, sg = blockIdx.x % q.n_seg, seq = row / c.n_kv;
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int32_t* kr = kept + (size_t)row * q.budget;
    const int s0 = min(len, sg * q.seg), s1 = min(len, s0 + q.seg);
    if (bad || len <= q.budget) {
        if (LEVEL == 3) {
            if (bad && tid == 0) raise_table();
            for (int i = sg * kSelThreads + tid; i < q.budget; i += q.n_seg * kSelThreads) kr[i] = !bad && i < len ? i : -1;
        }
        return;
    }
    const int z = len - q.recent, segs = (len + q.seg - 1) / q.seg;
    if (sg >= segs) return;
    const float* wr = w + (size_t)row * c.max_pages * kPage;
    uint32_t need = q.budget - q.sink - q.recent, cut = 0;
    const bool choose = need > 0;
    uint32_t* const h0 = q.hist + (size_t)row * 3 * kSegs * kBins;
    uint32_t* const ab = q.above + (size_t)row * 2 * kSegs;
    uint32_t* const st = q.state + (size_t)row * 4;
    int low_before = 0;                                  // ranks of earlier segments that the low bits put above the cut
    if (LEVEL > 0 && choose) {
        if (LEVEL > 1) {
            cut = st[2 * (LEVEL - 2)];
            need = st[2 * (LEVEL - 2) + 1];
        }
        const int hi = kBins - 2 * (tid + 1);
        const uint32_t* hl = h0 + (size_t)(LEVEL - 1) * kSegs * kBins + hi;
        uint32_t lo = 0, up = 0, lo_b = 0, up_b = 0;
        if (LEVEL < 3 || hi < 1024)                      // the low bits have 1024 bins
            for (int s0 = 0; s0 < segs; s0 += 16) {      // slots behind the last segment are there, and not counted
                uint2 x[16];
#pragma unroll
                for (int s = 0; s < 16; s++) x[s] = *(const uint2*)(hl + (size_t)(s0 + s) * kBins);
#pragma unroll
                for (int s = 0; s < 16; s++) {
                    const bool in = s0 + s < segs, before = s0 + s < sg;
                    lo += in ? x[s].x : 0u;
                    up += in ? x[s].y : 0u;
                    if (LEVEL == 3) {
                        lo_b += before ? x[s].x : 0u;
                        up_b += before ? x[s].y : 0u;
                    }
                }
            }
        const uint32_t bin = pick_bin(bp, lo, up, need);
        cut |= bin << bin_shift(LEVEL - 1);
        if (LEVEL == 3) low_before = (hi > (int)bin ? lo_b : 0u) + (hi + 1 > (int)bin ? up_b : 0u);
        else if (sg == 0 && tid == 0) {
            st[2 * (LEVEL - 1)] = cut;
            st[2 * (LEVEL - 1) + 1] = need;
        }
    }
    if constexpr (LEVEL < 3) {
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        constexpr uint32_t known = LEVEL == 0 ? 0u : LEVEL == 1 ? ~0u << 21 : ~0u << 10;
        constexpr uint32_t group = LEVEL <= 1 ? 0u : ~0u << 21;   // bits that the launch before knew
        int over = 0;
#pragma unroll 4
        for (int i0 = s0 + wave * 64; i0 < s1; i0 += kSelThreads) {
            const int i = i0 + lane;
            const bool cand = i < s1 && i >= q.sink && i < z && choose;
            const uint32_t r = cand ? rank_of(wr[i]) : 0u;
            if (cand && (r & known) == cut) atomicAdd(&hist[bin_of(r, LEVEL)], 1u);
            if (LEVEL > 0) over += __popcll(__ballot(cand && (r & known) > cut && (r & group) == (cut & group)));
        }
        if (LEVEL > 0 && lane == 0) cnt2[wave][0] = over;
        __syncthreads();
        uint32_t* ho = h0 + ((size_t)LEVEL * kSegs + sg) * kBins;
        for (int i = tid; i < (LEVEL == 2 ? 1024 : kBins); i += kSelThreads) ho[i] = hist[i];
        if (LEVEL > 0 && tid == 0) {
            int sum = 0;
            for (int k = 0; k < kSelWaves; k++) sum += cnt2[k][0];
            ab[(LEVEL - 1) * kSegs + sg] = sum;
        }
    } else {
        // what the segments before this one keep: all outside [sink, z), the
        // ranks above the cut, and the equal ones up to `need`
        int sure = 0, eqs = 0;
        if (lane < sg && choose) {                       // kSegs <= 64: every wavefront for itself
            sure = ab[lane] + ab[kSegs + lane];
            eqs = h0[((size_t)2 * kSegs + lane) * kBins + (cut & 1023)];
        }
        sure = wave_isum_dpp(sure);
        eqs = wave_isum_dpp(eqs);
        // this segment: each wavefront its stretch
        const int per = (q.seg + kSelWaves * 64 - 1) / (kSelWaves * 64) * 64;
        const int a = s0 + wave * per, e = min(s1, a + per);
        int above = 0, equal = 0;
#pragma unroll 4
        for (int i0 = a; i0 < e; i0 += 64) {
            const int i = i0 + lane;
            const bool in = i < e, cand = in && i >= q.sink && i < z;
            const uint32_t r = cand ? rank_of(wr[i]) : 0u;
            above += __popcll(__ballot(in && (!cand || (choose && r > cut))));
            equal += __popcll(__ballot(cand && choose && r == cut));
        }
        low_before = wave_isum_dpp(low_before);
        if (lane == 0) {
            cnt2[wave][0] = above;
            cnt2[wave][1] = equal;
            cnt2[wave][2] = low_before;
        }
        __syncthreads();
        int at = sure + min(s0, q.sink) + max(0, s0 - z);
        for (int k = 0; k < kSelWaves; k++) {
            at += cnt2[k][2];
            if (k < wave) {
                at += cnt2[k][0];
                eqs += cnt2[k][1];
            }
        }
        at += min(eqs, (int)need);
        const unsigned long long low = (1ull << lane) - 1;
#pragma unroll 4
        for (int i0 = a; i0 < e; i0 += 64) {
            const int i = i0 + lane;
            const bool in = i < e, cand = in && i >= q.sink && i < z;
            const uint32_t r = cand ? rank_of(wr[i]) : 0u;
            const bool eq = cand && choose && r == cut;
            const unsigned long long be = __ballot(eq);
            const bool keep = in && (!cand || (choose && r > cut) || (eq && eqs + __popcll(be & low) < (int)need));
            const unsigned long long bk = __ballot(keep);
            if (keep) kr[at + __popcll(bk & low)] = i;
            at += __popcll(bk);
            eqs += __popcll(be);
        }
    }
}

// Moves the kept positions.  A group of 128 HDG threads gathers a page of the
// destination into registers, 16 bytes of keys, one pair and 16 bytes of values
// a thread, and writes them; a block has GROUPS such groups.  Not in place
// (GROUPS 1) a block is one page.  In place a block takes all pages of its (KV
// head, sequence) in order, GROUPS at a time: a kept position never lies
// before its destination, so page p's sources are in pages >= p, and a page is
// written only after it and the pages before it have been gathered.
//
// Values: a lane's 16 bytes hold 16 positions of two dims, so they come from up
// to 16 places.  A load takes 16 lanes of each of four positions (those of one
// half of a word, 16 apart), 256 contiguous bytes each, of which one nibble a
// dim is used; the lanes then hand each other their nibbles (each half, then
// each quarter of the lanes keeps its share) and end with what they write.
// (Gathered byte by byte into LDS the page took 61 us where this takes 31: 16
// sequences of 8 heads of 128 cut to 2000 positions.)
template <int GROUPS, int HDG>
__global__ __launch_bounds__(128 * HDG * GROUPS, GROUPS == 1 ? 5 : 4) void kv4_move(Kv4 src, Kv4 dst, const float* w_src, float* w_dst,
                                                               int budget, const int32_t* __restrict__ kept) {
    constexpr int hd = 64 * HDG, TG = 128 * HDG;
    // of a position: where the pool holds its 16 dims 0 .. of keys, its pair
    // of dims 0 .., its quarter of the values' first chunk; and the mask and
    // place of its nibble in the 8 bytes of a dim (word, shift).  A position
    // that is not there reads the pool's first bytes, masked away, so that no
    // load stands behind a branch.
    __shared__ int64_t koff[GROUPS][kPage], poff[GROUPS][kPage], voff[GROUPS][kPage];
    __shared__ uint32_t there[GROUPS][kPage], lost[GROUPS][kPage], nib[GROUPS][kPage];
    __shared__ int first[GROUPS];
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = wv / (2 * HDG), wave = wv % (2 * HDG), lane = threadIdx.x & 63, tid = wave * 64 + lane;
    const int li = lane & 15, lq = lane >> 4;
    int b = blockIdx.x;
    const int p0 = GROUPS > 1 ? 0 : b % dst.max_pages;
    if (GROUPS == 1) b /= dst.max_pages;
    const int h = b % src.n_kv, seq = b / src.n_kv;
    const int32_t* kr = kept + ((size_t)seq * src.n_kv + h) * budget;
    const float* ws = w_src + ((size_t)seq * src.n_kv + h) * src.max_pages * kPage;
    float* wd = w_dst + ((size_t)seq * src.n_kv + h) * dst.max_pages * kPage;
    const int p1 = GROUPS > 1 ? dst.max_pages : p0 + 1;
    if (p0 == 0 && h == 0 && threadIdx.x == 0 && kr[0] < 0) dst.lens[seq] = 0;
    for (int pb = p0; pb < p1; pb += GROUPS) {
        const int p = pb + grp;
        float wt = 0.f;
        uint8_t* const to = p < p1 ? page_at(dst, seq, p, h) : nullptr;
        if (tid < kPage) {
            const int i = p * kPage + tid;
            const int f = p < p1 && i < budget ? kr[i] : -1;
            const uint8_t* pg = nullptr;
            if (f >= 0) {
                pg = page_at(src, seq, f / kPage, h);
                wt = ws[f];
                if (!pg || !to) raise_table();
                if (h == 0 && (i + 1 == budget || kr[i + 1] < 0)) dst.lens[seq] = i + 1;
            }
            const int s = f & 63;
            const int64_t at = pg ? pg - src.pool : 0;
            koff[grp][tid] = pg ? at + key_off(s, 0, 0, HDG) : 0;
            poff[grp][tid] = pg ? at + 32 * hd + 4 * slot_of(s) : 0;
            voff[grp][tid] = pg ? at + 36 * hd + (s & 15) / 4 * 256 : 0;
            there[grp][tid] = pg ? ~0u : 0u;
            lost[grp][tid] = f >= 0 && !pg ? 0x7e007e00u : 0u;
            nib[grp][tid] = ((s >> 1) & 1) * 32 + 8 * (s >> 4) + 4 * (s & 1);
            if (tid == 0) first[grp] = f;
        }
        __syncthreads();
        const bool some = first[grp] >= 0;
        uint4 kx = make_uint4(0u, 0u, 0u, 0u), vx = kx;
        uint32_t px = 0;
        if (some) {
            // values of dims 32 wave ..: positions 16 lq + 2 r + hl of word r, half hl
            u32x4_t x[8][2];
#pragma unroll
            for (int r = 0; r < 8; r++)
#pragma unroll
                for (int hl = 0; hl < 2; hl++)
                    x[r][hl] = *(const u32x4_t*)(src.pool + voff[grp][16 * lq + 2 * r + hl] + (there[grp][16 * lq + 2 * r + hl] & (wave * 1024 + li * 16)));
            // keys: 16 dims of positions 32 u + li and 32 u + 16 + li; pairs of side u
            const int g = wave % HDG, u = wave / HDG;
            uint2 y[2];
            uint32_t my[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int t = 32 * u + 16 * k + li;
                my[k] = there[grp][t];
                y[k] = *(const uint2*)(src.pool + koff[grp][t] + (my[k] & (g * 1024 + lq * 256)));
            }
            const uint32_t mp = there[grp][lane];
            const uint32_t pr = *(const uint32_t*)(src.pool + poff[grp][lane] + (mp & (36 * hd * u + g * 256)));
            // every load above is on its way before the first is used: the
            // compiler would otherwise take each apart, and wait, at once
#pragma unroll
            for (int r = 0; r < 8; r++)
#pragma unroll
                for (int hl = 0; hl < 2; hl++) asm volatile("" : "+v"(x[r][hl]));
            kx = make_uint4(y[0].x & my[0], y[0].y & my[0], y[1].x & my[1], y[1].y & my[1]);
            px = (pr & mp) | lost[grp][lane];
            // word r of the lane's dims li and 16 + li, byte lq
            uint32_t w0[8], w1[8];
#pragma unroll
            for (int r = 0; r < 8; r++) {
                w0[r] = w1[r] = 0;
#pragma unroll
                for (int hl = 0; hl < 2; hl++) {
                    const uint32_t s = nib[grp][16 * lq + 2 * r + hl], m = there[grp][16 * lq + 2 * r + hl] & 15u;
                    w0[r] |= (((s & 32) ? x[r][hl].y : x[r][hl].x) >> (s & 31) & m) << (8 * lq + 4 * hl);
                    w1[r] |= (((s & 32) ? x[r][hl].w : x[r][hl].z) >> (s & 31) & m) << (8 * lq + 4 * hl);
                }
            }
            // lanes 0 - 31 keep words 0 - 3, the others 4 - 7; then each 16 their two
            uint32_t a0[4], a1[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool up = lq >= 2;
                a0[i] = (up ? w0[4 + i] : w0[i]) | __shfl_xor(up ? w0[i] : w0[4 + i], 32, kWave);
                a1[i] = (up ? w1[4 + i] : w1[i]) | __shfl_xor(up ? w1[i] : w1[4 + i], 32, kWave);
            }
            uint32_t c0[2], c1[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const bool up = lq & 1;
                c0[i] = (up ? a0[2 + i] : a0[i]) | __shfl_xor(up ? a0[i] : a0[2 + i], 16, kWave);
                c1[i] = (up ? a1[2 + i] : a1[i]) | __shfl_xor(up ? a1[i] : a1[2 + i], 16, kWave);
            }
            vx = make_uint4(c0[0], c0[1], c1[0], c1[1]);
        }
        __syncthreads();
        if (some && to) {
            const int g = wave % HDG, u = wave / HDG;
            *(uint4*)(to + wave * 1024 + lane * 16) = kx;      // chunk (u, g) is number u HDG + g
            *(uint4*)(to + 36 * hd + wave * 1024 + lane * 16) = vx;
            ((uint32_t*)(to + (32 + 36 * u) * hd))[g * 64 + slot_of(lane)] = px;
        }
        if (tid < kPage && p < p1) wd[p * kPage + tid] = wt;
        if (GROUPS > 1) __syncthreads();
    }
}

// ── host side ────────────────────────────────────────────────────────────────
bool cache_ok(const ibh_kv4_cache* c, const char* who) {
    if (!c || !c->pool || !c->table || !c->lens || c->n_pages <= 0 || c->n_seq <= 0 || c->max_pages <= 0 ||
        c->max_pages > (1 << 24) || c->n_kv <= 0 || c->head_dim < 64 || c->head_dim > 256 || c->head_dim % 64 ||
        ((uintptr_t)c->pool & 15)) {
        if (!c) ibh_set_error("%s: no cache given", who);
        else
            ibh_set_error("%s: invalid cache (pages=%d seqs=%d max_pages=%d kv_heads=%d head_dim=%d; head_dim 64, 128, "
                          "192 or 256, a pool on 16 bytes)", who, c->n_pages, c->n_seq, c->max_pages, c->n_kv,
                          c->head_dim);
        return false;
    }
    return true;
}
Kv4 device_of(const ibh_kv4_cache* c) {
    return {(uint8_t*)c->pool, c->table, c->lens, c->n_pages, c->n_seq, c->max_pages, c->n_kv, c->head_dim};
}
// A launch takes less than 2^32 threads.
bool grid_ok(size_t blocks, size_t threads, const char* who) {
    if (blocks < ((size_t)1 << 32) / threads) return true;
    ibh_set_error("%s: %zu blocks of work are more than one launch takes", who, blocks);
    return false;
}

}  // namespace

void* ibh_workspace(size_t bytes);

int ibh_kv4_errors(bool clear) {
    unsigned int v = 0;
    if (hipMemcpyFromSymbol(&v, HIP_SYMBOL(ibh_kv4_err), sizeof(v)) != hipSuccess) return -1;
    if (clear && v) {
        const unsigned int z = 0;
        if (hipMemcpyToSymbol(HIP_SYMBOL(ibh_kv4_err), &z, sizeof(z)) != hipSuccess) return -1;
    }
    return (int)v;
}

extern "C" size_t ibh_kv4_page_bytes(int n_kv, int head_dim) {
    if (n_kv <= 0 || head_dim < 64 || head_dim > 256 || head_dim % 64) return 0;
    return (size_t)n_kv * 72 * head_dim;
}

extern "C" int ibh_kv4_append(const ibh_kv4_cache* cache, const float* k, const float* v, int n_new, int kv_stride,
                              void* stream) {
    if (!cache_ok(cache, "ibh_kv4_append")) return IBH_ERROR_PARAM;
    if (!k || !v || n_new <= 0 || kv_stride < cache->n_kv * cache->head_dim) {
        ibh_set_error("ibh_kv4_append: invalid arguments (n_new=%d kv_stride=%d)", n_new, kv_stride);
        return IBH_ERROR_PARAM;
    }
    const int n_touch = min((n_new + kPage - 2) / kPage + 1, cache->max_pages);
    const size_t blocks = (size_t)cache->n_seq * n_touch * cache->n_kv * 2 * (cache->head_dim / 64);
    if (!grid_ok(blocks, 256, "ibh_kv4_append")) return IBH_ERROR_PARAM;
    const int vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && kv_stride % 4 == 0;
    kv4_append_kernel<<<(unsigned)blocks, 256, 0, ibh_resolve_stream(stream)>>>(device_of(cache), k, v, n_new,
                                                                                kv_stride, n_touch, vec);
    IBH_CHECK_LAUNCH("ibh_kv4_append");
    return IBH_OK;
}

extern "C" int ibh_kv4_read(const ibh_kv4_cache* cache, float* k, float* v, int n, int kv_stride, void* stream) {
    if (!cache_ok(cache, "ibh_kv4_read")) return IBH_ERROR_PARAM;
    if (!k || !v || n <= 0 || kv_stride < cache->n_kv * cache->head_dim) {
        ibh_set_error("ibh_kv4_read: invalid arguments (n=%d kv_stride=%d)", n, kv_stride);
        return IBH_ERROR_PARAM;
    }
    const int n_touch = min((n + kPage - 2) / kPage + 1, cache->max_pages);
    const size_t blocks = (size_t)cache->n_seq * n_touch * cache->n_kv * 2 * (cache->head_dim / 64);
    if (!grid_ok(blocks, 256, "ibh_kv4_read")) return IBH_ERROR_PARAM;
    const int vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && kv_stride % 4 == 0;
    kv4_read_kernel<<<(unsigned)blocks, 256, 0, ibh_resolve_stream(stream)>>>(device_of(cache), k, v, n, kv_stride,
                                                                              n_touch, vec);
    IBH_CHECK_LAUNCH("ibh_kv4_read");
    return IBH_OK;
}

// How a call is cut: row tiles of 4 rt query rows, blocks of `chunk` pages.
struct AttnPlan {
    int rt, n_tile, n_split, chunk, quantum, nw;         // rt 16: kv4_attn_wide
    uint32_t per_split;
    bool joint;                                          // the weights in the launch that joins the splits
    size_t blocks, joins, weighs;                        // blocks of the launches: attention, joining splits (and joint weights), weights
    int weigh_nw;                                        // wavefronts of a block of the weights' launch
    size_t part, part_ml, stat, digits, rowc, score, bytes;     // offsets into the workspace
};
static AttnPlan attn_plan(const ibh_kv4_cache* c, int n_heads, int n_q, bool weights) {
    AttnPlan p;
    const size_t n_rows = (size_t)n_q * (n_heads / c->n_kv), hdg = c->head_dim / 64;
    const size_t heads = (size_t)c->n_seq * c->n_kv;
    // Few rows: the smallest tile that holds them, so that pages are read once.
    // A tile of 16 rows does not fit the registers with head_dim above 128: tiles
    // of 8 there.  From 33 rows on the f16 kernel: 8 sequences of 4096
    // positions, 8 KV heads of 128, 24 rows 34 us here and 37 there, 32 rows 37
    // and 39, 40 rows 58 and 39, 64 rows 57 and 42.  (One sequence, where neither
    // fills the card, is faster here: 40 rows 17 and 20, 64 rows 18 and 24.)
    const bool wide = n_rows > 32;
    p.rt = wide ? kWideRows / 4 : n_rows <= 4 ? 1 : n_rows <= 8 || hdg > 2 ? 2 : 4;
    p.n_tile = (int)((n_rows + 4 * p.rt - 1) / (4 * p.rt));
    const size_t base = heads * p.n_tile;
    p.nw = 4;
    p.quantum = 4;
    size_t n = 1;
    if (wide) {
        // every block works at once, or in whole rounds: what a round takes in
        // pages (and one for its start), and what the partial sums cost that
        // are written and joined (228 blocks' as much as a page, a launch 1.5:
        // fitted).  Times with no split, with the number that this takes and
        // with the best of 1 to 256: 512 queries of 8 x 4 heads of 128 over 4100
        // positions 163, 132, 127 us; 40 rows of 8 heads over 4096, one sequence
        // 135, 21, 18, eight 138, 40, 40, 32 of 2048 78, 67, 67; 72 rows of 4
        // heads of 64 in 8 sequences of 2049 47, 24, 22; 64 rows over 20000 676,
        // 34, 34.
        p.quantum = 1;
        const size_t slots = 256 * (hdg == 1 ? 3 : hdg == 2 ? 2 : 1);
        double least = (double)((base + slots - 1) / slots) * (c->max_pages + 1);
        for (size_t k = 1; k <= 4; k++) {
            const size_t m = min(min(k * slots / base, (size_t)c->max_pages), (size_t)kMaxSplit);
            if (m < 2) continue;
            const double cost = (double)((base * m + slots - 1) / slots) * ((c->max_pages + m - 1) / m + 1) + base * m / 228.0 + 1.5;
            if (cost < least) {
                least = cost;
                n = m;
            }
        }
    } else {
        // as many blocks as the card holds at once: each has its rows to set
        // up and its sums to write and join (8 sequences of 4096 positions, 8
        // KV heads of 128: 13 us with 4 rows, 37 with 32; 16 and 43 with 2048
        // and 1024 blocks where 768 and 512 are held)
        const size_t work = base * c->max_pages, want = 256 * attn_waves((int)hdg, p.rt);
        size_t chunk = (work + want - 1) / want;
        chunk = max(chunk, ((size_t)c->max_pages + kMaxSplit - 1) / kMaxSplit);
        chunk = (chunk + 3) / 4 * 4;
        // in tables of up to 1024 positions few rows are one launch: eight
        // wavefronts take a head's pages, and nothing is left to join (600
        // positions of 32/4 heads: 6.9 us, 8.5 by blocks of 4 pages and a join)
        if (p.n_tile == 1 && p.rt <= 2 && (int)hdg * p.rt <= 6 && c->max_pages > 4 && c->max_pages <= 16) {
            p.nw = 8;
            chunk = 16;
        }
        n = (c->max_pages + chunk - 1) / chunk;
    }
    p.n_split = (int)n;
    p.per_split = n > 1 ? (uint32_t)((((uint64_t)1 << 32) + n - 1) / n) : 0;
    p.chunk = n > 1 ? chunk_of(c->max_pages, p.n_split, p.per_split, p.quantum) : c->max_pages;
    p.joint = weights && p.n_tile == 1 && p.n_split > 1 && p.rt <= 2;
    p.blocks = base * p.n_split;
    const size_t all = heads * n_rows;
    p.joins = p.n_split == 1 ? 0 : wide && p.n_split <= kFewSplits ? (all + 3) / 4 : all;
    if (p.joint) p.joins += heads * ((c->max_pages + 3) / 4);
    p.weighs = weights && !p.joint ? heads * c->max_pages : 0;
    // Wavefronts a page.  Many rows: four, eight where there are few pages
    // (2048 rows, 8 KV heads of 128: 167 and 178 us with 512 pages, 81 and 65
    // with 80; 40 rows, 4096 pages: 63 and 92; whole calls).  Up to 32: one
    // where the pages fill the card or have few rows, else eight (24 rows: 46
    // and 59 us with 4096 pages, 19 and 17 with 80; 12 rows: 32 and 44, 17 and 16).
    if (wide) p.weigh_nw = p.weighs >= 512 ? 4 : 8;
    else p.weigh_nw = p.weighs >= 2048 || n_rows <= 16 ? 1 : 8;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
    p.part = take(p.n_split > 1 ? heads * n_rows * p.n_split * c->head_dim * sizeof(float) : 0);
    p.part_ml = take(p.n_split > 1 ? heads * n_rows * p.n_split * sizeof(float2) : 0);
    const size_t pad = wide ? (n_rows + kWideRows - 1) / kWideRows * kWideRows : n_rows;
    const size_t again = weights && !p.joint ? heads : 0;
    p.stat = take(again * pad * sizeof(float2));
    p.digits = take(again * ((pad + 3) / 4) * hdg * 1024);
    p.rowc = take(again * pad * (1 + hdg) * sizeof(float));
    p.score = take(p.joint ? heads * c->max_pages * p.rt * 1024 : 0);
    p.bytes = at;
    return p;
}

extern "C" size_t ibh_kv4_attn_workspace_bytes(const ibh_kv4_cache* cache, int n_heads, int n_q, int weights) {
    if (!cache || cache->n_seq <= 0 || cache->n_kv <= 0 || cache->max_pages <= 0 || cache->head_dim < 64 ||
        cache->head_dim > 256 || cache->head_dim % 64 || n_heads <= 0 || n_heads % cache->n_kv || n_q <= 0)
        return 0;
    return attn_plan(cache, n_heads, n_q, weights != 0).bytes;
}

template <int HDG, int RT>
static void launch_attn_rt(const Kv4& c, const AttnArgs& a, const AttnPlan& p, size_t heads, const float* win,
                           float* wout, hipStream_t st) {
    const unsigned blocks = (unsigned)p.blocks, weighs = (unsigned)p.weighs;
    if constexpr (RT <= 2) {
        if (p.joint) kv4_attn_kernel<HDG, RT, true, 4><<<blocks, 256, 0, st>>>(c, a);
        else if constexpr (HDG * RT <= 6) if (p.nw == 8) kv4_attn_kernel<HDG, RT, false, 8><<<blocks, 512, 0, st>>>(c, a);
    }
    if (!p.joint && p.nw == 4) kv4_attn_kernel<HDG, RT, false, 4><<<blocks, 256, 0, st>>>(c, a);
    const unsigned rows = p.n_split > 1 ? (unsigned)(heads * a.n_q * (a.n_heads / c.n_kv)) : 0;
    if (p.joins) kv4_attn_finish<HDG, (RT <= 2 ? RT : 1)><<<(unsigned)p.joins, 256, 0, st>>>(c, a, rows, win, wout);
    if (weighs && p.weigh_nw == 1) kv4_attn_weights<HDG, 1><<<weighs, 64, 0, st>>>(c, a, win, wout);
    else if (weighs) kv4_attn_weights<HDG, 8><<<weighs, 512, 0, st>>>(c, a, win, wout);
}
template <int HDG>
static void launch_attn(const Kv4& c, const AttnArgs& a, const AttnPlan& p, size_t heads, const float* win,
                        float* wout, hipStream_t st) {
    if (p.rt == kWideRows / 4) {
        const size_t rows = heads * a.n_q * (a.n_heads / c.n_kv), pad = heads * p.n_tile * kWideRows;
        const WideRows wr = wout ? WideRows{(h8_t*)a.digits, a.rowc, a.rowc + pad, a.stat} : WideRows{};
        kv4_attn_wide<HDG><<<(unsigned)p.blocks, 256, 0, st>>>(c, a, wr);
        if (p.n_split > kFewSplits) kv4_attn_finish<HDG, 1><<<(unsigned)p.joins, 256, 0, st>>>(c, a, (unsigned)rows, win, wout);
        else if (p.joins) kv4_attn_join<HDG><<<(unsigned)p.joins, 256, 0, st>>>(c, a, rows);
        if (p.weighs && p.weigh_nw == 4) kv4_weights_wide<HDG, 4><<<(unsigned)p.weighs, 256, 0, st>>>(c, a, wr, win, wout);
        else if (p.weighs) kv4_weights_wide<HDG, 8><<<(unsigned)p.weighs, 512, 0, st>>>(c, a, wr, win, wout);
    } else if (p.rt == 1) launch_attn_rt<HDG, 1>(c, a, p, heads, win, wout, st);
    else if (p.rt == 2) launch_attn_rt<HDG, 2>(c, a, p, heads, win, wout, st);
    else if constexpr (HDG <= 2) launch_attn_rt<HDG, 4>(c, a, p, heads, win, wout, st);
}

extern "C" int ibh_kv4_attn(const ibh_kv4_cache* cache, float* out, const float* q, int n_heads, int n_q, int q_stride,
                            const float* weights_in, float* weights_out, void* ws, size_t ws_bytes, void* stream) {
    if (!cache_ok(cache, "ibh_kv4_attn")) return IBH_ERROR_PARAM;
    if (!out || !q || n_heads <= 0 || n_heads % cache->n_kv || n_q <= 0 ||
        (int64_t)q_stride < (int64_t)n_heads * cache->head_dim || (int64_t)n_q * n_heads > 0x7fffffff / 16 ||
        !weights_in != !weights_out) {
        ibh_set_error("ibh_kv4_attn: invalid arguments (heads=%d/%d n_q=%d q_stride=%d; weights_in and weights_out "
                      "both or neither)", n_heads, cache->n_kv, n_q, q_stride);
        return IBH_ERROR_PARAM;
    }
    const AttnPlan p = attn_plan(cache, n_heads, n_q, weights_out != nullptr);
    if (!ws && p.bytes) {
        ws = ibh_workspace(p.bytes);
        ws_bytes = ws ? p.bytes : 0;
    }
    if (p.bytes && (!ws || ws_bytes < p.bytes || ((uintptr_t)ws & 15))) {
        ibh_set_error("ibh_kv4_attn: workspace of %zu bytes on 16 bytes needed", p.bytes);
        return IBH_ERROR_MEMORY;
    }
    const size_t heads = (size_t)cache->n_seq * cache->n_kv;
    if (!grid_ok(p.blocks, 64 * p.nw, "ibh_kv4_attn") || !grid_ok(p.joins, 256, "ibh_kv4_attn") ||
        !grid_ok(p.weighs, 64 * p.weigh_nw, "ibh_kv4_attn"))
        return IBH_ERROR_PARAM;
    char* w = (char*)ws;
    AttnArgs a{out, q, n_heads, n_q, q_stride, (float)(1.4426950408889634 / sqrt((double)cache->head_dim)),
               p.n_split, p.n_tile, p.chunk, p.quantum, p.per_split, 4 * p.rt, (float*)(w + p.part), (float2*)(w + p.part_ml),
               weights_out && !p.joint ? (float2*)(w + p.stat) : nullptr,
               p.rt == kWideRows / 4 ? p.n_tile * kWideRows : n_q * (n_heads / cache->n_kv),
               weights_out && !p.joint ? (i4_t*)(w + p.digits) : nullptr, (float*)(w + p.rowc), (float4*)(w + p.score)};
    const Kv4 c = device_of(cache);
    hipStream_t st = ibh_resolve_stream(stream);
    switch (cache->head_dim / 64) {
        case 1: launch_attn<1>(c, a, p, heads, weights_in, weights_out, st); break;
        case 2: launch_attn<2>(c, a, p, heads, weights_in, weights_out, st); break;
        case 3: launch_attn<3>(c, a, p, heads, weights_in, weights_out, st); break;
        default: launch_attn<4>(c, a, p, heads, weights_in, weights_out, st); break;
    }
    IBH_CHECK_LAUNCH("ibh_kv4_attn");
    return IBH_OK;
}

template <int HDG>
static void launch_move(const Kv4& s, const Kv4& d, const float* ws, float* wd, int budget, const int32_t* kept,
                        bool in_place, size_t blocks, hipStream_t st) {
    constexpr int G = 1024 / (128 * HDG);
    if (in_place) kv4_move<G, HDG><<<(unsigned)blocks, 128 * HDG * G, 0, st>>>(s, d, ws, wd, budget, kept);
    else kv4_move<1, HDG><<<(unsigned)blocks, 128 * HDG, 0, st>>>(s, d, ws, wd, budget, kept);
}
static bool select_in_one(const ibh_kv4_cache* c) { return (int64_t)c->max_pages * kPage <= kSelMost; }

extern "C" size_t ibh_kv4_evict_workspace_bytes(const ibh_kv4_cache* cache) {
    if (!cache || cache->n_seq <= 0 || cache->n_kv <= 0 || cache->max_pages <= 0 || select_in_one(cache)) return 0;
    return (size_t)cache->n_seq * cache->n_kv * (kSegs * (3 * kBins + 2) + 4) * sizeof(uint32_t);
}

extern "C" int ibh_kv4_evict(const ibh_kv4_cache* src, const ibh_kv4_cache* dst, const float* weights_src,
                             float* weights_dst, int budget, int sink, int recent, int32_t* kept, void* ws,
                             size_t ws_bytes, void* stream) {
    if (!cache_ok(src, "ibh_kv4_evict (from)") || !cache_ok(dst, "ibh_kv4_evict (to)")) return IBH_ERROR_PARAM;
    if (!weights_src || !weights_dst || !kept || budget <= 0 || sink < 0 || recent < 0 || sink > budget ||
        recent > budget - sink || (size_t)budget > (size_t)dst->max_pages * kPage || src->n_seq != dst->n_seq ||
        src->n_kv != dst->n_kv || src->head_dim != dst->head_dim) {
        ibh_set_error("ibh_kv4_evict: invalid arguments (budget=%d sink=%d recent=%d; sink + recent <= budget <= 64 "
                      "pages of the destination's rows, both caches of the same sequences, heads and head_dim)",
                      budget, sink, recent);
        return IBH_ERROR_PARAM;
    }
    const bool in_place = src->table == dst->table;
    if (in_place ? (src->pool != dst->pool || src->max_pages != dst->max_pages || src->lens != dst->lens || weights_src != weights_dst)
                 : (weights_src == weights_dst || src->lens == dst->lens)) {
        ibh_set_error("ibh_kv4_evict: in place takes the same pool, table, lens and weights on both sides; else all but "
                      "the pool differ");
        return IBH_ERROR_PARAM;
    }
    const size_t need = ibh_kv4_evict_workspace_bytes(src);
    if (!ws && need) {
        ws = ibh_workspace(need);
        ws_bytes = ws ? need : 0;
    }
    if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15))) {
        ibh_set_error("ibh_kv4_evict: workspace of %zu bytes on 16 bytes needed", need);
        return IBH_ERROR_MEMORY;
    }
    const size_t heads = (size_t)src->n_seq * src->n_kv;
    const size_t blocks = heads * (in_place ? 1 : dst->max_pages);
    if (!grid_ok(blocks, in_place ? 1024 : 2 * src->head_dim, "ibh_kv4_evict") ||
        !grid_ok(heads * (need ? kSegs : 1), kSelThreads, "ibh_kv4_evict"))
        return IBH_ERROR_PARAM;
    hipStream_t st = ibh_resolve_stream(stream);
    const Kv4 s = device_of(src), d = device_of(dst);
    if (!need) {
        if (src->max_pages * kPage <= 4 * kSelThreads)
            kv4_select<4><<<(unsigned)heads, kSelThreads, 0, st>>>(s, weights_src, budget, sink, recent, kept);
        else
            kv4_select<16><<<(unsigned)heads, kSelThreads, 0, st>>>(s, weights_src, budget, sink, recent, kept);
    } else {
        LongSel q;
        q.hist = (uint32_t*)ws;
        q.above = q.hist + heads * 3 * kSegs * kBins;
        q.state = q.above + heads * 2 * kSegs;
        // at least 4096 positions a segment: shorter ones cost more in adding up counts than they save
        q.seg = max(4096, ((src->max_pages + kSegs - 1) / kSegs) * kPage);
        q.n_seg = (int)(((int64_t)src->max_pages * kPage + q.seg - 1) / q.seg);
        q.budget = budget;
        q.sink = sink;
        q.recent = recent;
        const unsigned grid = (unsigned)(heads * q.n_seg);
        kv4_select_long<0><<<grid, kSelThreads, 0, st>>>(s, q, weights_src, kept);
        kv4_select_long<1><<<grid, kSelThreads, 0, st>>>(s, q, weights_src, kept);
        kv4_select_long<2><<<grid, kSelThreads, 0, st>>>(s, q, weights_src, kept);
        kv4_select_long<3><<<grid, kSelThreads, 0, st>>>(s, q, weights_src, kept);
    }
    IBH_CHECK_LAUNCH("ibh_kv4_evict (select)");
    switch (src->head_dim / 64) {
        case 1: launch_move<1>(s, d, weights_src, weights_dst, budget, kept, in_place, blocks, st); break;
        case 2: launch_move<2>(s, d, weights_src, weights_dst, budget, kept, in_place, blocks, st); break;
        case 3: launch_move<3>(s, d, weights_src, weights_dst, budget, kept, in_place, blocks, st); break;
        default: launch_move<4>(s, d, weights_src, weights_dst, budget, kept, in_place, blocks, st); break;
    }
    IBH_CHECK_LAUNCH("ibh_kv4_evict (move)");
    return IBH_OK;
}
