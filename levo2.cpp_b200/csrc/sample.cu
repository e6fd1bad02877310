// Next-token sampling from one given uniform number a row: temperature, top-k,
// top-p and min-p over logits that the penalty and the ignore list of the greedy
// selection have gone through (the formulas stand at levo_sampling).
//
// All three filters keep a prefix of one order (larger logit first, equal logits
// by index), and the draw is a place in that prefix.  So nothing is sorted: each
// is the search for the value v at which a running count or a running weight
// reaches a target, and for the place among the logits equal to v.  A kept set is
// "every logit above `value`, and the first `ties` equal to it".
//
// Weights are F64 exponentials rounded to multiples of 2^-44 of the largest and
// summed as 64-bit integers (131072 * 2^44 = 2^61): exact, in any order.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace levo {
namespace {

constexpr int kThreads = 512;
constexpr int kBins = 256;
constexpr int64_t kMaxVocab = int64_t(1) << 17;

struct SampleArgs {
    const void *logits;
    int64_t rows, vocab, ld;
    const float *uniforms, *temperature_rows, *top_p_rows, *min_p_rows;
    const int64_t *top_k_rows;
    float temperature, top_p, min_p, penalty;
    int64_t top_k;
    const int64_t *recent;
    int64_t recent_len, limit;
    const int64_t *ignore;
    int64_t n_ignore, streams;
    int64_t *out;
    float *logprob;
    int32_t *status;
};

__device__ __forceinline__ float load_logit(const float *p, int64_t i) { return p[i]; }
__device__ __forceinline__ float load_logit(const __half *p, int64_t i) { return __half2float(p[i]); }
__device__ __forceinline__ float load_logit(const __nv_bfloat16 *p, int64_t i) { return __bfloat162float(p[i]); }

// Integers in the order of the values (-0 and +0 are made one before).
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

// exp((v - top) / T) in units of 2^-44: 2^x, x = (v - top) * log2(e)/T in F64, as
// 2^n (n the nearest integer) times the Taylor series of 2^f, |f| <= 1/2, to
// degree 10 (the first term left out is (ln2/2)^11 / 11! = 2.2e-13).
constexpr double kLn2 = 0.693147180559945309417;
constexpr double ln2_coefficient(int k) {
    double c = 1.0;
    for (int i = 1; i <= k; ++i) c *= kLn2 / i;
    return c;
}

__device__ __forceinline__ unsigned long long weight_of(float v, float top, double scale) {
    if (v == top) return 1ull << 44;
    const double x = (static_cast<double>(v) - static_cast<double>(top)) * scale;
    if (!(x > -46.0)) return 0;
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
    const double r = x + kRound;
    const double f = x - (r - kRound);
    double p = ln2_coefficient(10);
#pragma unroll
    for (int k = 9; k >= 0; --k) p = __fma_rn(p, f, ln2_coefficient(k));
    // p * 2^(44 + n) <= 2^44: adding 2^52 rounds it to an integer in the low mantissa bits
    const double scaled = __hiloint2double(__double2hiint(p) + ((__double2loint(r) + 44) << 20), __double2loint(p));
    return static_cast<unsigned long long>(__double_as_longlong(scaled + 4503599627370496.0)) & ((1ull << 52) - 1);
}

struct Kept {
    uint32_t key;  // every logit with a larger key is kept, and the first `ties` with this one
    int64_t ties;
};

struct Found {
    uint32_t key;
    unsigned long long above;  // weight or count of what lies before this key's ties
    int64_t group;             // ties of this key that the kept set holds
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
    extern __shared__ uint32_t bits[];  // [pen words][ign words]
    __shared__ unsigned long long mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ unsigned long long total;
    __shared__ uint32_t top_key;
    __shared__ int nan_seen;
    __shared__ Found found;
    __shared__ int warp_count[kThreads / 32];
    __shared__ int64_t token;
    const int64_t words = (a.vocab + 31) / 32;
    uint32_t *pen = bits, *ign = bits + words;
    const int tid = threadIdx.x;

    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.logits) + row * a.ld;
        const bool ignores = a.ignore && (a.streams > 0 ? row % a.streams == 0 : row == 0);
        __syncthreads();
        for (int64_t w = tid; w < 2 * words; w += kThreads) bits[w] = 0u;
        if (tid == 0) {
            top_key = 0;
            nan_seen = 0;
        }
        __syncthreads();
        if (a.recent)
            for (int64_t j = tid; j < a.recent_len; j += kThreads) {
                const int64_t t = a.recent[row * a.recent_len + j];
                if (t >= 0 && t < a.limit) atomicOr(&pen[t >> 5], 1u << (t & 31));
            }
        if (ignores)
            for (int64_t j = tid; j < a.n_ignore; j += kThreads) {
                const int64_t t = a.ignore[j];
                if (t >= 0 && t < a.vocab) atomicOr(&ign[t >> 5], 1u << (t & 31));
            }
        __syncthreads();
        // The logit as the order sees it: NaN and ignored ids as -inf, -0 as +0.
        auto logit = [&](int64_t i) {
            float v = load_logit(x, i);
            const uint32_t m = 1u << (i & 31);
            if (pen[i >> 5] & m) v = __fdiv_rn(v, a.penalty);
            if (ign[i >> 5] & m) v = -INFINITY;
            if (isnan(v)) {
                nan_seen = 1;
                v = -INFINITY;
            }
            return v + 0.0f;
        };
        uint32_t best = 0;
        for (int64_t i = tid; i < a.vocab; i += kThreads) best = max(best, key_of(logit(i)));
        atomicMax(&top_key, best);
        __syncthreads();
        const float top = value_of(top_key);

        // this row's settings
        bool bad = false;
        float temperature = a.temperature_rows ? a.temperature_rows[row] : a.temperature;
        if (!(temperature >= 0.0f) || isinf(temperature)) bad = true, temperature = 0.0f;
        int64_t k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
        if (k < 0) bad = true, k = 0;
        if (k == 0 || k > a.vocab) k = a.vocab;
        float top_p = a.top_p_rows ? a.top_p_rows[row] : a.top_p;
        if (!(top_p >= 0.0f && top_p <= 1.0f)) bad = true, top_p = top_p < 0.0f ? 0.0f : 1.0f;
        float min_p = a.min_p_rows ? a.min_p_rows[row] : a.min_p;
        if (!(min_p >= 0.0f && min_p <= 1.0f)) bad = true, min_p = min_p > 1.0f ? 1.0f : 0.0f;
        float u = a.uniforms[row];
        if (!(u >= 0.0f && u < 1.0f)) bad = true, u = u >= 1.0f ? 1.0f : 0.0f;
        if (temperature == 0.0f) k = 1;
        const double scale = temperature > 0.0f ? 1.4426950408889634074 / static_cast<double>(temperature) : 0.0;
        const unsigned long long least =
            static_cast<unsigned long long>(ceil(static_cast<double>(min_p) * 17592186044416.0));  // 2^44

        // The key at which the running count (or weight) of the kept set first reaches `target`, eight bits a level.
        auto search = [&](const Kept &kept, bool by_weight, unsigned long long target) {
            uint32_t prefix = 0;
            unsigned long long above = 0;
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int j = tid; j < kBins; j += kThreads) mass[j] = 0, count[j] = 0;
                __syncthreads();
                auto add = [&](uint32_t key, uint32_t n) {
                    if (shift < 24 && (key >> (shift + 8)) != prefix) return;
                    const int bin = (key >> shift) & (kBins - 1);
                    atomicAdd(&count[bin], n);
                    if (by_weight) atomicAdd(&mass[bin], n * weight_of(value_of(key), top, scale));
                };
                for (int64_t i = tid; i < a.vocab; i += kThreads) {
                    const float v = logit(i);
                    if (v > -INFINITY && key_of(v) > kept.key) add(key_of(v), 1);
                }
                if (tid == 0 && kept.ties > 0) add(kept.key, static_cast<uint32_t>(kept.ties));
                __syncthreads();
                if (tid == 0) {
                    int bin = kBins - 1;
                    int last = -1;
                    for (; bin >= 0; --bin) {
                        const unsigned long long n = by_weight ? mass[bin] : count[bin];
                        if (count[bin]) last = bin;
                        if (above + n >= target && count[bin]) break;
                        if (bin) above += n;
                    }
                    if (bin < 0) bin = last;
                    found = {(prefix << 8) | static_cast<uint32_t>(bin), above, static_cast<int64_t>(count[bin])};
                }
                __syncthreads();
                prefix = found.key;
                above = found.above;
                __syncthreads();
            }
            return Found{prefix, above, found.group};
        };

        if (top == -INFINITY) {
            if (tid == 0) {
                a.out[row] = 0;
                if (a.logprob) a.logprob[row] = -INFINITY;
                if (a.status) atomicOr(a.status, LEVO_SAMPLE_EMPTY | (nan_seen ? LEVO_SAMPLE_NAN : 0) | (bad ? LEVO_SAMPLE_PARAM : 0));
            }
            continue;
        }
        Kept kept{key_of(-INFINITY), 0};
        if (k < a.vocab) {
            int64_t finite = 0;
            if (tid == 0) total = 0;
            __syncthreads();
            for (int64_t i = tid; i < a.vocab; i += kThreads) finite += logit(i) > -INFINITY;
            atomicAdd(&total, static_cast<unsigned long long>(finite));
            __syncthreads();
            const int64_t all = static_cast<int64_t>(total);
            __syncthreads();
            if (k < all) {
                const Found f = search(kept, false, static_cast<unsigned long long>(k));
                kept = {f.key, k - static_cast<int64_t>(f.above)};
            }
        }
        // weight of the kept set (of those at least `least`)
        auto weigh = [&](unsigned long long floor) {
            if (tid == 0) total = 0;
            __syncthreads();
            unsigned long long sum = 0;
            for (int64_t i = tid; i < a.vocab; i += kThreads) {
                const float v = logit(i);
                if (key_of(v) <= kept.key || v == -INFINITY) continue;
                const unsigned long long w = weight_of(v, top, scale);
                if (w >= floor) sum += w;
            }
            if (tid == 0 && kept.ties > 0) {
                const unsigned long long w = weight_of(value_of(kept.key), top, scale);
                if (w >= floor) sum += w * kept.ties;
            }
            atomicAdd(&total, sum);
            __syncthreads();
            const unsigned long long all = total;
            __syncthreads();
            return all;
        };
        unsigned long long weight = 0;
        if (top_p < 1.0f) {
            const double part = ceil(static_cast<double>(top_p) * static_cast<double>(weigh(0)));
            const unsigned long long target = max(1ull, static_cast<unsigned long long>(part));
            const Found f = search(kept, true, target);
            const unsigned long long w = max(1ull, weight_of(value_of(f.key), top, scale));
            const int64_t need = static_cast<int64_t>((target - f.above + w - 1) / w);
            kept = {f.key, min(f.group, max(need, int64_t(1)))};
        }
        weight = weigh(least);
        const unsigned long long target =
            min(static_cast<unsigned long long>(static_cast<double>(u) * static_cast<double>(weight)), weight - 1);
        const Found f = search(kept, true, target + 1);
        const unsigned long long w = max(1ull, weight_of(value_of(f.key), top, scale));
        const int64_t place = min(static_cast<int64_t>((target - f.above) / w), f.group - 1);
        // the place-th index whose logit has that key
        int64_t before = 0;
        for (int64_t i0 = 0; i0 < a.vocab; i0 += kThreads) {
            const int64_t i = i0 + tid;
            const bool is = i < a.vocab && key_of(logit(i)) == f.key;
            const uint32_t vote = __ballot_sync(0xffffffffu, is);
            if ((tid & 31) == 0) warp_count[tid >> 5] = __popc(vote);
            __syncthreads();
            int64_t mine = before + __popc(vote & ((1u << (tid & 31)) - 1));
            int64_t all = 0;
            for (int j = 0; j < kThreads / 32; ++j) {
                if (j < (tid >> 5)) mine += warp_count[j];
                all += warp_count[j];
            }
            if (is && mine == place) token = i;
            before += all;
            __syncthreads();
            if (before > place) break;
        }
        if (tid == 0) {
            a.out[row] = token;
            if (a.logprob)
                a.logprob[row] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(weight)));
            const int flags = (nan_seen ? LEVO_SAMPLE_NAN : 0) | (bad ? LEVO_SAMPLE_PARAM : 0);
            if (a.status && flags) atomicOr(a.status, flags);
        }
    }
}

template <typename T>
int launch_sample(const SampleArgs &a, const char *what, cudaStream_t stream) {
    const size_t smem = static_cast<size_t>(2 * ((a.vocab + 31) / 32)) * sizeof(uint32_t);
    const int64_t grid = std::min<int64_t>(a.rows, static_cast<int64_t>(sm_count()) * 4);
    sample_kernel<T><<<static_cast<unsigned>(grid), kThreads, smem, stream>>>(a);
    return check_launch(what);
}

}  // namespace
}  // namespace levo

extern "C" {

LEVO_OPS_API int levo_sample_tokens(const levo_sampling *sampling, levo_stream_t stream) {
    using namespace levo;
    clear_error();
    const char *w = "levo_sample_tokens";
    auto fail = [&](const char *why) { return set_error(LEVO_OPS_EINVAL, std::string(w) + why); };
    if (sampling == nullptr) return fail(": arguments are null");
    const levo_sampling &s = *sampling;
    size_t element = 0;
    switch (s.dtype) {
        case LEVO_DTYPE_F32: element = 4; break;
        case LEVO_DTYPE_F16:
        case LEVO_DTYPE_BF16: element = 2; break;
        default: return fail(": dtype must be F32, F16 or BF16");
    }
    if (s.rows < 0 || s.vocab < 0 || s.recent_len < 0 || s.n_ignore < 0 || s.streams < 0) return fail(": negative size");
    if (s.rows == 0) return LEVO_OPS_OK;
    if (s.vocab == 0) return fail(": cannot sample an empty vocabulary");
    if (s.vocab > kMaxVocab) return set_error(LEVO_OPS_EUNSUPPORTED, std::string(w) + ": vocabulary above 131072");
    if (s.ld < s.vocab) return fail(": row stride smaller than the vocabulary");
    if (s.logits == nullptr || s.uniforms == nullptr || s.tokens_out == nullptr) return fail(": required pointer is null");
    if (s.temperature_rows == nullptr && !(s.temperature >= 0.0f && std::isfinite(s.temperature)))
        return fail(": temperature must be finite and not negative");
    if (s.top_k_rows == nullptr && s.top_k < 0) return fail(": top_k must not be negative");
    if (s.top_p_rows == nullptr && !(s.top_p >= 0.0f && s.top_p <= 1.0f)) return fail(": top_p must lie in [0, 1]");
    if (s.min_p_rows == nullptr && !(s.min_p >= 0.0f && s.min_p <= 1.0f)) return fail(": min_p must lie in [0, 1]");
    if (s.recent != nullptr && s.recent_len > 0 && (!(s.penalty > 0.0f) || !std::isfinite(s.penalty)))
        return fail(": repetition penalty must be finite and positive");
    if (s.n_ignore > 0 && s.ignore == nullptr) return fail(": ignore list is null");
    const struct {
        const void *p;
        size_t align;
    } ptrs[] = {{s.logits, element}, {s.uniforms, 4}, {s.temperature_rows, 4}, {s.top_k_rows, 8}, {s.top_p_rows, 4},
                {s.min_p_rows, 4}, {s.recent, 8}, {s.ignore, 8}, {s.tokens_out, 8}, {s.logprob_out, 4}, {s.status, 4}};
    for (const auto &p : ptrs)
        if (p.p && !aligned_to(p.p, p.align)) return fail(": pointer is not aligned to its element size");
    const int64_t limit = s.penalty_limit <= 0 ? s.vocab : std::min(s.penalty_limit, s.vocab);
    const SampleArgs a{s.logits, s.rows, s.vocab, s.ld, s.uniforms, s.temperature_rows, s.top_p_rows, s.min_p_rows,
                       s.top_k_rows, s.temperature, s.top_p, s.min_p, s.penalty, s.top_k,
                       s.recent_len > 0 ? s.recent : nullptr, s.recent_len, limit,
                       s.n_ignore > 0 ? s.ignore : nullptr, s.n_ignore, s.streams, s.tokens_out, s.logprob_out,
                       s.status};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (s.dtype == LEVO_DTYPE_F32) return launch_sample<float>(a, w, st);
    if (s.dtype == LEVO_DTYPE_F16) return launch_sample<__half>(a, w, st);
    return launch_sample<__nv_bfloat16>(a, w, st);
}

}  // extern "C"
