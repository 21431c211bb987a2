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

// A sequence's length; one outside its table row is cut to it and reported.
__device__ __forceinline__ int seq_len(const Kv4& c, int seq, bool* bad) {
    const int n = c.lens[seq], cap = c.max_pages * kPage;
    const int m = n < 0 ? 0 : (n > cap ? cap : n);
    *bad = m != n;
    return m;
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
// (t, c) holds dims 16 i + 4 c .. + 3.  The group's ends give scale =
// f16((hi - lo) / 15) and mid = f16(lo + 8 scale); a code is the fp32 quotient
// rounded, then put right against the exact borders mid + (c +- 1/2) scale
// (fp64 holds both sides), so the codes are those of the exact quotient.
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4 c, const float* __restrict__ k,
                                                         const float* __restrict__ v, int n_new, int stride,
                                                         int n_touch, int vec) {
    __shared__ uint8_t code[kPage][68];
    const int hdg = c.hd / 64;
    int b = blockIdx.x;
    const int g = b % hdg; b /= hdg;
    const int side = b & 1; b >>= 1;
    const int h = b % c.n_kv; b /= c.n_kv;
    const int seq = b / n_touch;
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const int first = len - n_new;                       // position of row 0
    const int p = max(first, 0) / kPage + b % n_touch;
    if (bad) {
        if (threadIdx.x == 0) raise_table();
        return;
    }
    if (p * kPage >= len) return;
    uint8_t* const pg = page_at(c, seq, p, h);
    if (!pg) {
        if (threadIdx.x == 0) raise_table();
        return;
    }
    uint8_t* const part = pg + side * 36 * c.hd;
    const int tid = threadIdx.x, t = tid >> 2, cq = tid & 3;
    const int pos = p * kPage + t;
    const bool is_new = pos >= first && pos < len;
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
    float lo = INFINITY, hi = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        nan |= x[i] != x[i];
        x[i] = fminf(fmaxf(x[i], -65504.f), 65504.f);
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
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
    uint32_t word[4];                                    // four codes, a byte each
#pragma unroll
    for (int i = 0; i < 4; i++) {
        word[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float q = 0.f;
            if (sc > 0.f) {
                q = fminf(fmaxf(rintf((x[4 * i + j] - mid) / sc), -8.f), 7.f);
                const double d = (double)x[4 * i + j] - (double)mid;
                const double up = (double)((q + 0.5f) * sc), dn = (double)((q - 0.5f) * sc);
                const bool odd = ((int)q & 1) != 0;      // a tie goes to the even neighbour
                if (q < 7.f && (d > up || (d == up && odd))) q += 1.f;
                else if (q > -8.f && (d < dn || (d == dn && odd))) q -= 1.f;
            }
            word[i] |= (uint32_t)((int)q + 8) << (8 * j);
        }
    }
    if (side == 0) {
        // dims 16 i + 4 cq ..: word cq / 2 of block i, half cq % 2
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t o = __shfl_xor(word[i], 1, kWave);
            if (is_new && !(cq & 1)) *(uint32_t*)(part + key_off(t, g, i, hdg) + (cq >> 1) * 4) = word[i] | (o << 4);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) *(uint32_t*)&code[t][16 * i + 4 * cq] = word[i];
    __syncthreads();
    // a word of values holds eight positions of one dim: those that are not
    // new keep their nibbles (no other block writes this word)
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int d = tid & 63, r = (tid >> 6) + 4 * u;
        uint32_t w = 0, m = 0;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int hl = 0; hl < 2; hl++) {
                const int tt = 16 * i + 2 * r + hl, ps = p * kPage + tt;
                w |= (uint32_t)code[tt][d] << (8 * i + 4 * hl);
                if (ps >= first && ps < len) m |= 0xfu << (8 * i + 4 * hl);
            }
        if (!m) continue;
        uint32_t* dst = (uint32_t*)(part + val_off(64 * g + d, r));
        *dst = m == 0xffffffffu ? w : ((w & m) | (*dst & ~m));
    }
}

// ── read ─────────────────────────────────────────────────────────────────────
// The values of a sequence's last n positions: block as above.
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4 c, float* __restrict__ k, float* __restrict__ v, int n,
                                                       int stride, int n_touch) {
    const int hdg = c.hd / 64;
    int b = blockIdx.x;
    const int g = b % hdg; b /= hdg;
    const int side = b & 1; b >>= 1;
    const int h = b % c.n_kv; b /= c.n_kv;
    const int seq = b / n_touch;
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const int first = len - n;
    const int p = max(first, 0) / kPage + b % n_touch;
    if (bad && threadIdx.x == 0) raise_table();
    if (p * kPage >= len) return;
    const uint8_t* const pg = page_at(c, seq, p, h);
    if (!pg && threadIdx.x == 0) raise_table();
    const int tid = threadIdx.x, d = tid & 63;
    for (int t = tid >> 6; t < kPage; t += 4) {
        const int pos = p * kPage + t;
        if (pos < first || pos >= len) continue;
        float y = NAN;
        if (pg && !bad) {
            const uint8_t* part = pg + side * 36 * c.hd;
            const uint32_t pr = ((const uint32_t*)(part + 32 * c.hd))[g * 64 + slot_of(t)];
            int cd;
            if (side == 0) {
                const int e = d & 15;
                cd = part[key_off(t, g, d >> 4, hdg) + (e >> 3) * 4 + (e & 3)] >> (e & 4) & 15;
            } else {
                cd = part[val_off(64 * g + d, (t & 15) >> 1) + (t >> 4)] >> (4 * (t & 1)) & 15;
            }
            y = fmaf(h2f(pr), (float)(cd - 8), h2f(pr >> 16));
        }
        (side ? v : k)[((size_t)seq * n + (pos - first)) * (size_t)stride + h * c.hd + 64 * g + d] = y;
    }
}

// ── attention ────────────────────────────────────────────────────────────────
// Block (head, query, sequence): one pass over the pages with the running
// maximum and sum; the row's maximum and sum go to `stat` for the weights.
__global__ __launch_bounds__(256) void kv4_attn_rows(Kv4 c, float* __restrict__ out, const float* __restrict__ q,
                                                     int n_heads, int n_q, int q_stride, float scale,
                                                     float2* __restrict__ stat) {
    __shared__ float qs[256], sc[kPage], sv[kPage][4], mv[kPage][4], red[2];
    int b = blockIdx.x;
    const int hq = b % n_heads; b /= n_heads;
    const int qi = b % n_q, seq = b / n_q;
    const int hdg = c.hd / 64, h = hq / (n_heads / c.n_kv);
    const int tid = threadIdx.x;
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const int n = max(0, len - n_q + qi + 1);            // positions that this query sees
    if (tid < c.hd) qs[tid] = q[((size_t)seq * n_q + qi) * (size_t)q_stride + hq * c.hd + tid];
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int p = 0; p * kPage < n; p++) {
        const uint8_t* pg = page_at(c, seq, p, h);
        if (!pg) { bad = true; break; }
        const int t = tid >> 2, cq = tid & 3;
        __syncthreads();
        float s = 0.f;
        for (int g = 0; g < hdg; g++) {
            const uint32_t pr = ((const uint32_t*)(pg + 32 * c.hd))[g * 64 + slot_of(t)];
            const uint8_t* kb = pg + key_off(t, g, cq, hdg);
            const float ks = h2f(pr), km = h2f(pr >> 16);
            for (int e = 0; e < 16; e++) {
                const int cd = kb[(e >> 3) * 4 + (e & 3)] >> (e & 4) & 15;
                s = fmaf(qs[64 * g + 16 * cq + e], fmaf(ks, (float)(cd - 8), km), s);
            }
        }
        s += __shfl_xor(s, 1, kWave);
        s += __shfl_xor(s, 2, kWave);
        if (cq == 0) sc[t] = p * kPage + t < n ? s * scale : -INFINITY;
        if (cq < hdg) {
            const uint32_t pr = ((const uint32_t*)(pg + 68 * c.hd))[cq * 64 + slot_of(t)];
            sv[t][cq] = h2f(pr);
            mv[t][cq] = h2f(pr >> 16);
        }
        __syncthreads();
        if (tid < 64) {
            const float x = sc[tid];
            const float mn = fmaxf(m, wave_max(x));      // at least one position of the page is seen
            const float e = x == -INFINITY ? 0.f : expf(x - mn);
            const float a = expf(m - mn);
            l = l * a + wave_sum(e);
            m = mn;
            sc[tid] = e;
            if (tid == 0) red[0] = a;
        }
        __syncthreads();
        if (tid < c.hd) {
            o *= red[0];
            for (int tt = 0; tt < min(kPage, n - p * kPage); tt++) {
                const int cd = pg[36 * c.hd + val_off(tid, (tt & 15) >> 1) + (tt >> 4)] >> (4 * (tt & 1)) & 15;
                o = fmaf(sc[tt], fmaf(sv[tt][tid >> 6], (float)(cd - 8), mv[tt][tid >> 6]), o);
            }
        }
    }
    if (tid == 0) {
        red[0] = l;
        if (bad) raise_table();
        if (stat) stat[((size_t)seq * n_q + qi) * n_heads + hq] = bad ? make_float2(0.f, NAN) : make_float2(m, l);
    }
    __syncthreads();
    if (tid < c.hd)
        out[(((size_t)seq * n_q + qi) * n_heads + hq) * c.hd + tid] = bad ? NAN : (n ? o / red[0] : 0.f);
}

// Accumulated weights: block (page, KV head, sequence) scores its 64 positions
// again for every row of the head and adds e^(s - m) / l.
__global__ __launch_bounds__(256) void kv4_attn_weights(Kv4 c, const float* __restrict__ q, int n_heads, int n_q,
                                                        int q_stride, float scale, const float2* __restrict__ stat,
                                                        const float* __restrict__ win, float* __restrict__ wout) {
    int b = blockIdx.x;
    const int p = b % c.max_pages; b /= c.max_pages;
    const int h = b % c.n_kv, seq = b / c.n_kv;
    const int hdg = c.hd / 64, grp = n_heads / c.n_kv;
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const int t = threadIdx.x >> 2, cq = threadIdx.x & 3, pos = p * kPage + t;
    const size_t at = ((size_t)seq * c.n_kv + h) * c.max_pages * kPage + pos;
    float acc = 0.f;
    if (p * kPage < len) {
        const uint8_t* pg = page_at(c, seq, p, h);
        bad |= !pg;
        for (int r = 0; pg && r < n_q * grp; r++) {
            const int qi = r / grp, hq = h * grp + r % grp;
            if (p * kPage > len - n_q + qi) continue;
            const float* qr = q + ((size_t)seq * n_q + qi) * (size_t)q_stride + hq * c.hd;
            float s = 0.f;
            for (int g = 0; g < hdg; g++) {
                const uint32_t pr = ((const uint32_t*)(pg + 32 * c.hd))[g * 64 + slot_of(t)];
                const uint8_t* kb = pg + key_off(t, g, cq, hdg);
                const float ks = h2f(pr), km = h2f(pr >> 16);
                for (int e = 0; e < 16; e++) {
                    const int cd = kb[(e >> 3) * 4 + (e & 3)] >> (e & 4) & 15;
                    s = fmaf(qr[64 * g + 16 * cq + e], fmaf(ks, (float)(cd - 8), km), s);
                }
            }
            s += __shfl_xor(s, 1, kWave);
            s += __shfl_xor(s, 2, kWave);
            const float2 ml = stat[((size_t)seq * n_q + qi) * n_heads + hq];
            if (pos <= len - n_q + qi) acc += expf(s * scale - ml.x) / ml.y;
        }
    }
    if (cq == 0) wout[at] = pos < len ? (bad ? NAN : win[at] + acc) : 0.f;
}

// ── eviction ─────────────────────────────────────────────────────────────────
// Order-preserving integer of a weight: NaN lowest, -0 and +0 alike.
__device__ __forceinline__ uint32_t rank_of(float w) {
    if (w != w) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;

// Block (KV head, sequence): the need-th largest weight of positions
// [sink, len - recent) byte by byte from the top (a histogram of the ranks
// that share the bytes found so far), then the kept positions in order:
// wavefront w counts and then emits its own stretch of the positions.
__global__ __launch_bounds__(kSelThreads) void kv4_select(Kv4 c, const float* __restrict__ w, int budget, int sink,
                                                          int recent, int32_t* __restrict__ kept) {
    __shared__ unsigned hist[256];
    __shared__ unsigned pick[2];
    __shared__ int cnt[kSelWaves][2];
    const int seq = blockIdx.x / c.n_kv;
    bool bad;
    const int len = seq_len(c, seq, &bad);
    const float* wr = w + (size_t)blockIdx.x * c.max_pages * kPage;
    int32_t* kr = kept + (size_t)blockIdx.x * budget;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (bad && tid == 0) raise_table();
    if (bad || len <= budget) {
        for (int i = tid; i < budget; i += kSelThreads) kr[i] = !bad && i < len ? i : -1;
        return;
    }
    const int z = len - recent;                          // candidates [sink, z)
    unsigned need = budget - sink - recent, prefix = 0, mask = 0;
    for (int shift = 24; need && shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = sink + tid; i < z; i += kSelThreads) {
            const uint32_t r = rank_of(wr[i]);
            if ((r & mask) == prefix) atomicAdd(&hist[(r >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            unsigned left = need;
            int d = 255;
            for (; d > 0 && hist[d] < left; d--) left -= hist[d];
            pick[0] = d;
            pick[1] = left;
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        mask |= 255u << shift;
        need = pick[1];
    }
    // kept: rank above the prefix, and the first `need` of those equal to it
    const bool none = budget == sink + recent;
    const int per = (len + kSelWaves * 64 - 1) / (kSelWaves * 64) * 64;
    const int a = wave * per, e = min(len, a + per);
    int above = 0, equal = 0;
    for (int i0 = a; i0 < e; i0 += 64) {
        const int i = i0 + lane;
        const bool cand = i < e && i >= sink && i < z;
        const uint32_t r = cand ? rank_of(wr[i]) : 0u;
        const bool sure = i < e && (!cand || (!none && r > prefix));
        const bool eq = cand && !none && r == prefix;
        above += __popcll(__ballot(sure));
        equal += __popcll(__ballot(eq));
    }
    if (lane == 0) { cnt[wave][0] = above; cnt[wave][1] = equal; }
    __syncthreads();
    int at = 0, eqs = 0;                                 // kept entries and equal ranks before this stretch
    for (int k = 0; k < wave; k++) {
        at += cnt[k][0];
        eqs += cnt[k][1];
    }
    at += min(eqs, (int)need);
    for (int i0 = a; i0 < e; i0 += 64) {
        const int i = i0 + lane;
        const bool cand = i < e && i >= sink && i < z;
        const uint32_t r = cand ? rank_of(wr[i]) : 0u;
        const bool eq = cand && !none && r == prefix;
        const unsigned long long be = __ballot(eq), low = (1ull << lane) - 1;
        const bool keep = i < e && (!cand || (!none && r > prefix) || (eq && eqs + __popcll(be & low) < (int)need));
        const unsigned long long bk = __ballot(keep);
        if (keep) kr[at + __popcll(bk & low)] = i;
        at += __popcll(bk);
        eqs += __popcll(be);
    }
}

// Moves the kept positions: block (first page, KV head, sequence) gathers a
// page of the destination into LDS and writes it.  In place (`serial`) a block
// takes all pages of its head in order: a kept position never lies before its
// destination, so page p's sources are in pages >= p, and page p is written
// only after pages <= p have been gathered.
__global__ __launch_bounds__(256) void kv4_move(Kv4 src, Kv4 dst, const float* w_src, float* w_dst, int budget,
                                                const int32_t* __restrict__ kept, int serial) {
    extern __shared__ __align__(16) uint8_t buf[];       // 72 hd bytes
    __shared__ int from[kPage];
    __shared__ float wt[kPage];
    const int hd = src.hd, hdg = hd / 64, tid = threadIdx.x;
    int b = blockIdx.x;
    const int p0 = serial ? 0 : b % dst.max_pages;
    if (!serial) b /= dst.max_pages;
    const int h = b % src.n_kv, seq = b / src.n_kv;
    const int32_t* kr = kept + ((size_t)seq * src.n_kv + h) * budget;
    const float* ws = w_src + ((size_t)seq * src.n_kv + h) * src.max_pages * kPage;
    float* wd = w_dst + ((size_t)seq * src.n_kv + h) * dst.max_pages * kPage;
    if (tid == 0 && p0 == 0 && h == 0 && kr[0] < 0) dst.lens[seq] = 0;
    const int p1 = serial ? dst.max_pages : p0 + 1;
    for (int p = p0; p < p1; p++) {
        __syncthreads();
        if (tid < kPage) {
            const int i = p * kPage + tid;
            const int f = i < budget ? kr[i] : -1;
            from[tid] = f;
            wt[tid] = f >= 0 ? ws[f] : 0.f;
            if (h == 0 && f >= 0 && (i + 1 == budget || kr[i + 1] < 0)) dst.lens[seq] = i + 1;
        }
        __syncthreads();
        if (from[0] >= 0) {
            bool bad = false;
            // keys: 8-byte pieces (position, 16 dims); pairs of both sides
            for (int i = tid; i < kPage * hdg * 4; i += 256) {
                const int t = i & 63, pc = i >> 6, f = from[t];
                uint2 x = make_uint2(0u, 0u);
                if (f >= 0) {
                    const uint8_t* pg = page_at(src, seq, f / kPage, h);
                    if (pg) x = *(const uint2*)(pg + key_off(f & 63, pc >> 2, pc & 3, hdg));
                }
                *(uint2*)(buf + key_off(t, pc >> 2, pc & 3, hdg)) = x;
            }
            for (int i = tid; i < kPage * hdg * 2; i += 256) {
                const int t = i & 63, g = (i >> 6) % hdg, side = (i >> 6) / hdg, f = from[t];
                uint32_t x = 0;
                if (f >= 0) {
                    const uint8_t* pg = page_at(src, seq, f / kPage, h);
                    bad |= !pg;
                    x = pg ? ((const uint32_t*)(pg + (32 + 36 * side) * hd))[g * 64 + slot_of(f & 63)] : 0x7e007e00u;
                }
                ((uint32_t*)(buf + (32 + 36 * side) * hd))[g * 64 + slot_of(t)] = x;
            }
            // values: a word of eight positions of one dim
            for (int i = tid; i < hd * 8; i += 256) {
                const int d = i % hd, r = i / hd;
                uint32_t x = 0;
                for (int k = 0; k < 8; k++) {
                    const int t = 16 * (k >> 1) + 2 * r + (k & 1), f = from[t];
                    if (f < 0) continue;
                    const uint8_t* pg = page_at(src, seq, f / kPage, h);
                    if (!pg) continue;
                    const uint32_t cd = pg[36 * hd + val_off(d, (f & 15) >> 1) + ((f & 63) >> 4)] >> (4 * (f & 1)) & 15;
                    x |= cd << (8 * (k >> 1) + 4 * (k & 1));
                }
                *(uint32_t*)(buf + 36 * hd + val_off(d, r)) = x;
            }
            if (bad) raise_table();
        }
        __syncthreads();
        if (from[0] >= 0) {
            uint8_t* pg = page_at(dst, seq, p, h);
            if (pg) {
                for (int i = tid; i < 72 * hd / 16; i += 256) ((uint4*)pg)[i] = ((const uint4*)buf)[i];
            } else if (tid == 0) {
                raise_table();
            }
        }
        if (tid < kPage) wd[p * kPage + tid] = wt[tid];
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
bool grid_ok(size_t blocks, const char* who) {
    if (blocks <= 0x7fffffffu) return true;
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
    if (!grid_ok(blocks, "ibh_kv4_append")) return IBH_ERROR_PARAM;
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
    if (!grid_ok(blocks, "ibh_kv4_read")) return IBH_ERROR_PARAM;
    kv4_read_kernel<<<(unsigned)blocks, 256, 0, ibh_resolve_stream(stream)>>>(device_of(cache), k, v, n, kv_stride,
                                                                              n_touch);
    IBH_CHECK_LAUNCH("ibh_kv4_read");
    return IBH_OK;
}

extern "C" size_t ibh_kv4_attn_workspace_bytes(const ibh_kv4_cache* cache, int n_heads, int n_q) {
    if (!cache || cache->n_seq <= 0 || n_heads <= 0 || n_q <= 0) return 0;
    return (size_t)cache->n_seq * n_q * n_heads * sizeof(float2);
}

extern "C" int ibh_kv4_attn(const ibh_kv4_cache* cache, float* out, const float* q, int n_heads, int n_q, int q_stride,
                            const float* weights_in, float* weights_out, void* ws, size_t ws_bytes, void* stream) {
    if (!cache_ok(cache, "ibh_kv4_attn")) return IBH_ERROR_PARAM;
    if (!out || !q || n_heads <= 0 || n_heads % cache->n_kv || n_q <= 0 || (size_t)q_stride < (size_t)n_heads * cache->head_dim ||
        !weights_in != !weights_out) {
        ibh_set_error("ibh_kv4_attn: invalid arguments (heads=%d/%d n_q=%d q_stride=%d; weights_in and weights_out "
                      "both or neither)", n_heads, cache->n_kv, n_q, q_stride);
        return IBH_ERROR_PARAM;
    }
    const size_t need = ibh_kv4_attn_workspace_bytes(cache, n_heads, n_q);
    if (!ws) {
        ws = ibh_workspace(need);
        ws_bytes = ws ? need : 0;
    }
    if (!ws || ws_bytes < need || ((uintptr_t)ws & 15)) {
        ibh_set_error("ibh_kv4_attn: workspace of %zu bytes on 16 bytes needed", need);
        return IBH_ERROR_MEMORY;
    }
    const size_t rows = (size_t)cache->n_seq * n_q * n_heads;
    const size_t wb = (size_t)cache->n_seq * cache->n_kv * cache->max_pages;
    if (!grid_ok(rows, "ibh_kv4_attn") || !grid_ok(wb, "ibh_kv4_attn")) return IBH_ERROR_PARAM;
    const float scale = 1.0f / sqrtf((float)cache->head_dim);
    hipStream_t st = ibh_resolve_stream(stream);
    float2* stat = (float2*)ws;
    kv4_attn_rows<<<(unsigned)rows, 256, 0, st>>>(device_of(cache), out, q, n_heads, n_q, q_stride, scale, stat);
    IBH_CHECK_LAUNCH("ibh_kv4_attn");
    if (weights_out) {
        kv4_attn_weights<<<(unsigned)wb, 256, 0, st>>>(device_of(cache), q, n_heads, n_q, q_stride, scale, stat,
                                                       weights_in, weights_out);
        IBH_CHECK_LAUNCH("ibh_kv4_attn (weights)");
    }
    return IBH_OK;
}

extern "C" int ibh_kv4_evict(const ibh_kv4_cache* src, const ibh_kv4_cache* dst, const float* weights_src,
                             float* weights_dst, int budget, int sink, int recent, int32_t* kept, void* stream) {
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
    const size_t heads = (size_t)src->n_seq * src->n_kv;
    const size_t blocks = heads * (in_place ? 1 : dst->max_pages);
    if (!grid_ok(blocks, "ibh_kv4_evict")) return IBH_ERROR_PARAM;
    hipStream_t st = ibh_resolve_stream(stream);
    kv4_select<<<(unsigned)heads, kSelThreads, 0, st>>>(device_of(src), weights_src, budget, sink, recent, kept);
    IBH_CHECK_LAUNCH("ibh_kv4_evict (select)");
    kv4_move<<<(unsigned)blocks, 256, 72 * src->head_dim, st>>>(device_of(src), device_of(dst), weights_src,
                                                                weights_dst, budget, kept, in_place ? 1 : 0);
    IBH_CHECK_LAUNCH("ibh_kv4_evict (move)");
    return IBH_OK;
}
