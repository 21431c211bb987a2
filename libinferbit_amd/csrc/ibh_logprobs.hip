// ibh_logprobs.hip -- log-probabilities of given tokens, entropy and the best
// alternatives of rows of logits.
#include "ibh_common.h"

namespace {
using namespace ibh;

constexpr int kT = 1024;

struct LogArgs {
    float *out, *entropy, *top_lp;
    int32_t* top_ids;
    const float* z;
    const int32_t* tokens;
    int V, n_tok, k;
    size_t stride;
};

// A logit and its place as one whole number: larger is better, of equal logits
// the lower place.
__device__ __forceinline__ uint64_t key_of(float z, int id) {
    uint32_t b = __builtin_bit_cast(uint32_t, z + 0.f);  // -0 ties with 0
    b = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)b << 32 | (uint32_t)~id;
}

__global__ __launch_bounds__(kT) void logprobs_kernel(LogArgs a) {
    __shared__ float sm[kT / 64], ss[kT / 64], se[kT / 64];
    __shared__ uint64_t sk[kT / 64];
    const size_t row = blockIdx.x;
    const float* z = a.z + row * a.stride;
    const int tid = threadIdx.x, wave = tid >> 6;
    float m = -__builtin_inff();
    bool nan = false;
    for (int j = tid; j < a.V; j += kT) {
        nan |= !(z[j] < __builtin_inff());
        m = fmaxf(m, z[j]);
    }
    m = wave_max(nan ? __builtin_inff() : m);
    if ((tid & 63) == 0) sm[wave] = m;
    __syncthreads();
    for (int i = 0; i < kT / 64; i++) m = fmaxf(m, sm[i]);
    float s = 0, e = 0;
    for (int j = tid; j < a.V; j += kT) {
        const float d = z[j] - m, p = expf(d);
        if (z[j] > -__builtin_inff()) s += p, e += p * d;
    }
    s = wave_sum(s);
    e = wave_sum(e);
    if ((tid & 63) == 0) ss[wave] = s, se[wave] = e;
    __syncthreads();
    s = e = 0;
    for (int i = 0; i < kT / 64; i++) s += ss[i], e += se[i];
    const bool bad = m == __builtin_inff(), none = m == -__builtin_inff();
    const float lse = logf(s), nanf = __builtin_nanf("");
    for (int t = tid; t < a.n_tok; t += kT) {
        const int id = a.tokens[row * a.n_tok + t];
        a.out[row * a.n_tok + t] = bad || id < 0 || id >= a.V ? nanf : none ? -__builtin_inff() : (z[id] - m) - lse;
    }
    if (a.entropy && tid == 0) a.entropy[row] = bad ? nanf : none ? 0.f : lse - e / s;
    uint64_t last = ~0ull;
    for (int t = 0; t < a.k; t++) {
        uint64_t best = 0;
        if (!bad)
            for (int j = tid; j < a.V; j += kT) {
                const uint64_t key = key_of(z[j], j);
                if (z[j] > -__builtin_inff() && key < last && key > best) best = key;
            }
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor(best, o, 64);
            best = other > best ? other : best;
        }
        if ((tid & 63) == 0) sk[wave] = best;
        __syncthreads();
        for (int i = 0; i < kT / 64; i++) best = sk[i] > best ? sk[i] : best;
        __syncthreads();
        const int id = ~(uint32_t)best;
        if (tid == 0) {
            a.top_ids[row * a.k + t] = best ? id : -1;
            a.top_lp[row * a.k + t] = bad ? nanf : best ? (z[id] - m) - lse : -__builtin_inff();
        }
        last = best;
    }
}

}  // namespace

extern "C" size_t ibh_logprobs_workspace_bytes(int V, int B, int k) { return 0; }

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
    if (B >= (1 << 22)) {
        ibh_set_error("ibh_logprobs: %d rows are more than one launch takes", B);
        return IBH_ERROR_PARAM;
    }
    const LogArgs a{out, entropy, top_logprobs, top_ids, logits, tokens, V, n_tokens, k, (size_t)stride};
    logprobs_kernel<<<B, kT, 0, ibh_resolve_stream(stream)>>>(a);
    IBH_CHECK_LAUNCH("ibh_logprobs");
    return IBH_OK;
}
