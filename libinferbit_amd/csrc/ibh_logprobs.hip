// ibh_logprobs.hip -- log-probabilities of given tokens, entropy and the best
// alternatives of rows of logits.
//
// One pass over a row: every lane keeps the running maximum m, s = sum e^(z - m)
// and e = sum e^(z - m) (z - m) of its logits, every wavefront the k best it has
// seen.  log S = m + log s; entropy = log s - e / s.
//
// Memory bounds long calls: 2047 rows of 32003, 262 MB, take 49 us without
// alternatives (5.3 TB/s, as a copy does), 59 with the 8 best and 67 with 20:
// the candidates' instructions (a wavefront's bar is the k-th best of its first
// 1024 logits, so each later piece has about k).  Short calls are chains: of 32 x
// 128000 with the 20 best, 11.3 us in the first launch and 4.9 in the one that joins
// the shares, half of the first one's blocks are done after 7.4 us (their last logits
// there 3.3, candidates held 4.6, the block's wavefronts there 5.6, their sums joined
// 5.8, their lists sorted 7.1), the last after 9.9.  (Kernels, traced one by one; a
// row of calls with the 8 best takes 57 us each.)
#include "ibh_common.h"

namespace {
using namespace ibh;

constexpr int kWaves = 4, kManyWaves = 16;               // of a block
constexpr int kPiece = 1024;                             // logits that a wavefront takes at a time
constexpr int kHeld = 256;                               // candidates that it holds
constexpr int kManyRows = 256;                           // that fill the card by themselves
constexpr int kMaxShares = 64;                          // blocks that share a row, at most
constexpr float kLog2e = 1.44269504088896340736f;

typedef float f4_t __attribute__((ext_vector_type(4), aligned(4)));

struct LogArgs {
    float *out, *entropy, *top_lp;
    int32_t* top_ids;
    const float* z;
    const int32_t* tokens;
    int V, n_tok, k;
    size_t stride;
    int S, seg;                                          // blocks that share a row, logits of each
    float* part;                                         // [B][S]{m, s, e, -}
    uint64_t* keys;                                      // [B][S][k], the best of each share, in no order, 0 behind them
};

// ── sums ─────────────────────────────────────────────────────────────────────
struct Sums {
    float m, s, e;                                       // s is NaN where a logit is NaN or +infinity
};
// What the sums of maximum `from` are multiplied by, and the distance, where
// the maximum becomes `to`.  Masked logits (-infinity) and empty sums come out
// as a factor of 0 beside a finite distance, so that no 0 * infinity arises.
__device__ __forceinline__ float down(float from, float to, float* d) {
    const float x = from - (to == -__builtin_inff() ? 0.f : to);
    *d = fmaxf(x, -1e4f);
    return __builtin_amdgcn_exp2f(x * kLog2e);
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    float da, db;
    const float fa = down(a.m, r.m, &da), fb = down(b.m, r.m, &db);
    r.s = a.s * fa + b.s * fb;
    r.e = fa * (a.e + a.s * da) + fb * (b.e + b.s * db);
    return r;
}
__device__ __forceinline__ Sums wave_join(Sums a) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        a = join(a, {__shfl_xor(a.m, o, kWave), __shfl_xor(a.s, o, kWave), __shfl_xor(a.e, o, kWave)});
    return a;
}

// ── the k best ───────────────────────────────────────────────────────────────
// A logit and its place as one whole number: larger is better, of equal logits
// the lower place.
__device__ __forceinline__ uint32_t order_of(float z) {
    const uint32_t b = __float_as_uint(z + 0.f);         // -0 ties with 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float z, int id) { return (uint64_t)order_of(z) << 32 | (uint32_t)~id; }
constexpr uint64_t kNothing = 0x007fffffffffffffull;     // -infinity: what is to be held has to be above

// A wavefront's candidates: at most kHeld keys, among them the k largest seen;
// keys up to `bar` are known not to be among them.
struct Best {
    uint64_t* held;
    int n, k;
    uint64_t bar;

    // Leaves the k largest, the largest first: each of up to 64 counts those
    // above it.
    __device__ __forceinline__ void sort() {
        if (n > 64) cut();
        const int lane = threadIdx.x & 63;
        const uint64_t mine = lane < n ? held[lane] : 0;
        int above = 0;
#pragma unroll 8
        for (int i = 0; i < n; i++) above += held[i] > mine;
        if (lane < n) held[above] = mine;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        n = n < k ? n : k;
    }
    // Leaves the k largest in any order: their smallest is found bit by bit.
    __device__ __forceinline__ void cut() {
        if (n <= k) return;
        const int lane = threadIdx.x & 63;
        uint64_t key[kHeld / 64];
#pragma unroll
        for (int i = 0; i < kHeld / 64; i++) key[i] = i * 64 + lane < n ? held[i * 64 + lane] : 0;
        uint64_t t = 0;
        for (int bit = 63; bit >= 0; bit--) {
            const uint64_t c = t | 1ull << bit;
            int above = 0;
#pragma unroll
            for (int i = 0; i < kHeld / 64; i++) above += __popcll(__ballot(key[i] >= c));
            if (above >= k) t = c;
            if (above == k) break;
        }
        int at = 0;
#pragma unroll
        for (int i = 0; i < kHeld / 64; i++) {
            const uint64_t keep = __ballot(key[i] >= t);
            if (key[i] >= t) held[at + __popcll(keep & ((1ull << lane) - 1))] = key[i];
            at += __popcll(keep);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        n = at;
        bar = t > bar ? t : bar;
    }
    __device__ __forceinline__ void offer(uint64_t key) {
        uint64_t more = __ballot(key > bar);
        if (!more) return;
        if (n + __popcll(more) > kHeld) {
            cut();
            more = __ballot(key > bar);
        }
        const int lane = threadIdx.x & 63;
        if (key > bar) held[n + __popcll(more & ((1ull << lane) - 1))] = key;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // other lanes read it
        n += __popcll(more);
    }
    // No logit below this one is above the bar, nor one of -infinity.
    __device__ __forceinline__ float least() const {
        const uint32_t o = (uint32_t)(bar >> 32);
        return fmaxf(__uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o), -3.40282347e38f);
    }
    // A bar to begin with, from the upper half of each lane's largest key: the
    // k-th largest of those (at least k keys are as large).
    __device__ __forceinline__ void first(uint32_t upper) {
        uint32_t t = 0;
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t c = t | 1u << bit;
            const int above = __popcll(__ballot(upper >= c));
            if (above >= k) t = c;
            if (above == k) break;
        }
        const uint64_t b = ((uint64_t)t << 32) - 1;
        if (t && b > bar) bar = b;
    }
};

template <int W>
struct Shared {
    uint64_t held[W][kHeld];
    int counts[W];
    Sums sums[W];
};

// The block's sums in every thread; its best, sorted, with the first wavefront.
template <int W>
__device__ __forceinline__ Sums gather(Sums t, Best& best, Shared<W>& sh) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    t = wave_join(t);
    if (best.n > 64) best.cut();
    if (lane == 0) sh.sums[wave] = t, sh.counts[wave] = best.n;
    __syncthreads();
    t = sh.sums[0];
    for (int w = 1; w < W; w++) t = join(t, sh.sums[w]);
    if (wave || !best.k) return t;
    uint64_t key[W], top = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        key[w] = lane < sh.counts[w] ? sh.held[w][lane] : 0;
        top = key[w] > top ? key[w] : top;
    }
    best.n = 0;
    best.bar = kNothing;
    best.first((uint32_t)(top >> 32));
#pragma unroll
    for (int w = 0; w < W; w++) best.offer(key[w]);
    best.sort();
    return t;
}

// The row's outputs.
template <int W>
__device__ __forceinline__ void finish(const LogArgs& a, size_t row, Sums t, const Best& best) {
    const int tid = threadIdx.x;
    const float* z = a.z + row * a.stride;
    const bool bad = t.s != t.s, none = t.m == -__builtin_inff();
    const float logs = logf(t.s), nanf = __builtin_nanf("");
    for (int i = tid; i < a.n_tok; i += W * 64) {
        const int id = a.tokens[row * a.n_tok + i];
        a.out[row * a.n_tok + i] = bad || id < 0 || id >= a.V ? nanf : none ? -__builtin_inff() : (z[id] - t.m) - logs;
    }
    if (a.entropy && tid == 0) a.entropy[row] = bad ? nanf : none ? 0.f : logs - t.e / t.s;
    if (tid >= a.k) return;
    const bool held = !bad && tid < best.n;              // fewer than k may be left
    const int id = held ? (int)~(uint32_t)best.held[tid] : -1;
    a.top_ids[row * a.k + tid] = id;
    a.top_lp[row * a.k + tid] = bad ? nanf : held ? (z[id] - t.m) - logs : -__builtin_inff();
}

template <int W>
__global__ __launch_bounds__(W * 64, W == kWaves ? 8 : 4) void logprobs_kernel(LogArgs a) {
    __shared__ Shared<W> sh;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const size_t row = blockIdx.x / a.S;
    const int share = blockIdx.x % a.S;
    const float* z = a.z + row * a.stride;
    // pieces begin on 16 bytes, up to three logits in front of a row that does not
    const int off = (int)((uintptr_t)z >> 2) & 3;
    const int v0 = share * a.seg - off, v1 = min(v0 + a.seg, a.V);
    Sums t{-__builtin_inff(), 0.f, 0.f};
    Best best{sh.held[wave], 0, a.k, kNothing};
    // one piece ahead; a piece that is not whole reads single logits, -infinity
    // for those outside the share
    f4_t next[4];
    bool begin = true;
    auto from = [&](int j) { return (const char*)z + (uint32_t)j * 4u; };    // V is at most 2^30
    for (int at = v0 + (wave - W) * kPiece; at < v1; at += W * kPiece) {
        f4_t v[4];
#pragma unroll
        for (int q = 0; q < 4; q++) v[q] = next[q];
        const int ahead = at + W * kPiece;
        if (ahead >= 0 && ahead + kPiece <= v1) {
#pragma unroll
            for (int q = 0; q < 4; q++) next[q] = *(const f4_t*)(from(ahead + lane * 4) + q * 1024);
        } else if (ahead < v1) {
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int j = ahead + q * 256 + lane * 4 + i;
                    const float x = *(const float*)from(min(max(j, 0), v1 - 1));
                    next[q][i] = j >= 0 && j < v1 ? x : -__builtin_inff();
                }
        }
        if (at < v0) continue;
        float top = v[0][0];
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) top = fmaxf(top, v[q][i]);
        float d;
        const float m = fmaxf(t.m, top), f = down(t.m, m, &d);
        Sums now{m, 0.f, 0.f};                           // apart, so that chains of additions stay short
        t = {m, t.s * f, f * (t.e + t.s * d)};
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = down(v[q][i], m, &d);
                now.s += p;
                now.e = fmaf(p, d, now.e);
            }
        t.s += now.s;
        t.e += now.e;
        if (!a.k) continue;
        const uint32_t o = order_of(top);
        if (begin) best.first(top > -__builtin_inff() ? o : 0);
        begin = false;
        if (!__ballot(o > (uint32_t)(best.bar >> 32))) continue;
        // each lane's own that may be above, one after the other (few: in
        // registers they are picked by halving, not by an index)
        const float least = best.least();
        uint32_t may = 0;
#pragma unroll
        for (int e = 0; e < 16; e++) may |= (uint32_t)(v[e / 4][e % 4] >= least) << e;
        for (; __ballot(may != 0); may &= may - 1) {
            const int e = may ? __ffs(may) - 1 : 0;
            const uint32_t s0 = -(uint32_t)(e & 1), s1 = -(uint32_t)(e >> 1 & 1), s2 = -(uint32_t)(e >> 2 & 1), s3 = -(uint32_t)(e >> 3);
            auto pick = [](uint32_t a, uint32_t b, uint32_t second) { return (a & ~second) | (b & second); };
            auto of4 = [&](f4_t w) {
                return pick(pick(__float_as_uint(w[0]), __float_as_uint(w[1]), s0),
                            pick(__float_as_uint(w[2]), __float_as_uint(w[3]), s0), s1);
            };
            const float x = __uint_as_float(pick(pick(of4(v[0]), of4(v[1]), s2), pick(of4(v[2]), of4(v[3]), s2), s3));
            best.offer(may ? key_of(x, at + e / 4 * 256 + lane * 4 + e % 4) : 0);
        }
    }
    t = gather(t, best, sh);
    if (a.S == 1) {
        finish<W>(a, row, t, best);
        return;
    }
    const size_t me = blockIdx.x;
    if (threadIdx.x == 0) *(f4_t*)(a.part + me * 4) = f4_t{t.m, t.s, t.e, 0.f};
    if ((int)threadIdx.x < a.k) a.keys[me * a.k + threadIdx.x] = lane < best.n ? best.held[lane] : 0;
}

// The shares of a row joined, by one wavefront: a few hundred keys, and all its
// time is the code that it has to fetch.
__global__ __launch_bounds__(64) void logprobs_join(LogArgs a) {
    __shared__ uint64_t held[kHeld];
    const int lane = threadIdx.x, n = a.S * a.k;
    const size_t row = blockIdx.x;
    const uint64_t* keys = a.keys + row * n;
    constexpr int kEach = 16;                            // keys of a lane under way at once
    uint64_t key[kEach];
    auto fetch = [&](int at) {
#pragma unroll
        for (int i = 0; i < kEach; i++) key[i] = at + i * 64 + lane < n ? keys[at + i * 64 + lane] : 0;
    };
    fetch(0);
    Sums t{-__builtin_inff(), 0.f, 0.f};
    if (lane < a.S) {
        const f4_t v = *(const f4_t*)(a.part + (row * a.S + lane) * 4);
        t = {v[0], v[1], v[2]};
    }
    t = wave_join(t);
    Best best{held, 0, a.k, kNothing};
    for (int at = 0; at < n; at += kEach * 64) {
        if (at) fetch(at);
        uint64_t top = 0;
#pragma unroll
        for (int i = 0; i < kEach; i++) top = key[i] > top ? key[i] : top;
        best.first((uint32_t)(top >> 32));
#pragma unroll
        for (int i = 0; i < kEach; i++)
            if (at + i * 64 < n) best.offer(key[i]);
    }
    best.sort();
    finish<1>(a, row, t, best);
}

// How a call is cut.  Rows that fill the card by themselves, and rows of one
// round of four wavefronts' pieces, take a block of four (300 x 128000, 20 best:
// 49 us, shared 38 + 5.3 in two launches, 60 in a block of sixteen, of which a CU
// holds one; 600 x 64000, 8 best: 40, 39 + 5.0 and 52).  Fewer rows of up to two
// rounds of sixteen take a block of those: one launch instead of two (1 x 32000, 5
// best: 10.3 us, shared 6.2 + 3.9; 255 rows, 20 best: 16 and 17 + 4.6; but 1 x 64000
// 14.6 and 6.2 + 3.9, 1 x 4000 7.6 and 6.2 in one block of four).  Otherwise a row
// is shared by blocks, whole rounds each, and the shares are joined (32 x 128000, 20
// best, 256, 512 and 1024 blocks in all: 13.7 + 4.7, 11.4 + 4.8 and 10.4 + 5.1; 8 x
// 260000, 256 and 512: 9.9 + 5.5 and 8.0 + 7.4).
struct LogPlan {
    int W, S, seg;
    size_t part, bytes;
};
LogPlan plan_of(int V, int B, int k) {
    LogPlan p;
    const bool one = V + 3 <= kWaves * kPiece;           // up to three in front of the row
    p.W = !one && B < kManyRows && V + 3 <= 2 * kManyWaves * kPiece ? kManyWaves : kWaves;
    const int round = p.W * kPiece, rounds = (V + 3 + round - 1) / round;
    const int want = p.W == kManyWaves || B >= kManyRows ? 1 : min(min(rounds, kMaxShares), (512 + B - 1) / B);
    const int each = (rounds + want - 1) / want;
    p.seg = each * round;
    p.S = (rounds + each - 1) / each;
    p.part = p.S > 1 ? (size_t)B * p.S * 16 : 0;
    p.bytes = p.S > 1 ? p.part + (size_t)B * p.S * k * 8 : 0;
    return p;
}

}  // namespace

void* ibh_workspace(size_t bytes);

extern "C" size_t ibh_logprobs_workspace_bytes(int V, int B, int k) {
    if (V <= 0 || V > (1 << 30) || B <= 0 || k < 0 || k > IBH_LOGPROBS_MAX_K) return 0;
    return plan_of(V, B, k).bytes;
}

extern "C" int ibh_logprobs(float* out, float* entropy, int32_t* top_ids, float* top_logprobs, const float* logits,
                            const int32_t* tokens, int V, int B, int stride, int n_tokens, int k, void* ws,
                            size_t ws_bytes, void* stream) {
    if (B == 0) return IBH_OK;
    if (!logits || V <= 0 || V > (1 << 30) || B < 0 || (B > 1 && stride < V) || n_tokens < 0 || k < 0 ||
        (n_tokens && (!out || !tokens)) || (k && (!top_ids || !top_logprobs)) || (!n_tokens && !k && !entropy)) {
        ibh_set_error("ibh_logprobs: invalid arguments (V=%d B=%d stride=%d n_tokens=%d k=%d; tokens with out, top_ids "
                      "with top_logprobs, an output at all)", V, B, stride, n_tokens, k);
        return IBH_ERROR_PARAM;
    }
    if (k > IBH_LOGPROBS_MAX_K) {
        ibh_set_error("ibh_logprobs: k=%d, at most %d", k, IBH_LOGPROBS_MAX_K);
        return IBH_ERROR_PARAM;
    }
    const size_t rows = B;
    const struct { const void* p; size_t n; } op[] = {{n_tokens ? out : nullptr, rows * n_tokens * 4}, {entropy, rows * 4},
        {k ? top_ids : nullptr, rows * k * 4}, {k ? top_logprobs : nullptr, rows * k * 4},
        {logits, ((rows - 1) * stride + V) * 4}, {n_tokens ? tokens : nullptr, rows * n_tokens * 4}};
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 6; j++)
            if (i != j && ibh_overlap(op[i].p, op[i].n, op[j].p, op[j].n)) {
                ibh_set_error("ibh_logprobs: an output overlaps another operand");
                return IBH_ERROR_PARAM;
            }
    const LogPlan p = plan_of(V, B, k);
    if ((size_t)B * p.S >= (1 << 24)) {                  // a launch takes less than 2^32 threads
        ibh_set_error("ibh_logprobs: %d rows are more than one launch takes", B);
        return IBH_ERROR_PARAM;
    }
    uint8_t* w = nullptr;
    if (p.bytes) {
        w = (uint8_t*)(ws ? (ws_bytes >= p.bytes && !((uintptr_t)ws & 15) ? ws : nullptr) : ibh_workspace(p.bytes));
        if (!w) {
            ibh_set_error("ibh_logprobs: a workspace of %zu bytes on 16 bytes is needed", p.bytes);
            return IBH_ERROR_MEMORY;
        }
    }
    const LogArgs a{out, entropy, top_logprobs, top_ids, logits, tokens, V, n_tokens, k, (size_t)stride, p.S, p.seg,
                    (float*)w, (uint64_t*)(w + p.part)};
    hipStream_t st = ibh_resolve_stream(stream);
    if (p.W == kWaves) logprobs_kernel<kWaves><<<B * p.S, kWaves * 64, 0, st>>>(a);
    else logprobs_kernel<kManyWaves><<<B * p.S, kManyWaves * 64, 0, st>>>(a);
    IBH_CHECK_LAUNCH("ibh_logprobs");
    if (p.S > 1) {
        logprobs_join<<<B, 64, 0, st>>>(a);
        IBH_CHECK_LAUNCH("ibh_logprobs");
    }
    return IBH_OK;
}
