// Next-token sampling from one given uniform number a row: temperature, top-k,
// top-p and min-p over logits that the penalty and the ignore list of the greedy
// selection have gone through (the formulas stand at levo_sampling).
//
// All three filters keep a prefix of one order (larger logit first, equal logits
// by index), and the draw is a place in that prefix.  So nothing is sorted: top-k,
// top-p and the draw are each the search for the one token at which a running
// count, or a running weight, passes a target:
//   1. a histogram (of counts, or of weights) over kBins equal slices of the
//      logits' range below the maximum, and its running sums;
//   2. the slice that the target falls into;
//   3. its tokens, some tens of 16385, in a list; each adds up what lies before it.
// A slice of more than kList tokens (many equal or close logits) is cut further by
// the bits of its keys until its tokens are few or all equal.
//
// Weights are F64 exponentials rounded to multiples of 2^-44 of the largest and
// summed as 64-bit integers (131072 * 2^44 = 2^61): exact, in any order, so that
// atomics and the split over CTAs cannot change a result.
//
// A row is held in shared memory as F32 and read from HBM once.  It is split over
// a cluster of up to 8 CTAs where there are few rows or it is long; the cluster's
// first CTA merges the histograms, takes the decisions and holds the list.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace levo {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 512;
constexpr int kMaxCluster = 8;
constexpr int kSearches = 16;  // lists of one row: three searches, each with up to three further cuts
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
    int chunk, slots;  // logits of a CTA, and its places in shared memory
};

// Integers in the order of the values (-0 and +0 are made one before).
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
// The order as one integer, ascending: larger logit first, then the smaller index.
__device__ __forceinline__ u64 order_of(float v, int index) {
    return (static_cast<u64>(~key_of(v)) << 32) | static_cast<uint32_t>(index);
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

// For v within 32 T of the top, as bin_of takes them: x > -47.
__device__ __forceinline__ u64 weight_of(float v, double top, double scale) {
    const double x = (static_cast<double>(v) - top) * scale;
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
    const double r = x + kRound;
    const double f = x - (r - kRound);
    double p = ln2_coefficient(10);
#pragma unroll
    for (int k = 9; k >= 0; --k) p = __fma_rn(p, f, ln2_coefficient(k));
    // p * 2^(44 + n) <= 2^44: adding 2^52 rounds it to an integer in the low mantissa bits
    const double scaled = __hiloint2double(__double2hiint(p) + ((__double2loint(r) + 44) << 20), __double2loint(p));
    return static_cast<u64>(__double_as_longlong(scaled + 4503599627370496.0)) & ((1ull << 52) - 1);
}

// A token found: its place in the order, what lies before it, and what it has itself (weight, or 1).
struct Found {
    u64 order, before, own;
};

struct Shared {
    u64 warp_sums[kWarps];
    u64 total;                        // first CTA: of the histogram
    u64 passing[kMaxCluster];         // first CTA: weight that min-p leaves, of each CTA
    Found found;
    u64 target;
    u64 before, upto;                 // the slice that the target falls into: what lies before it, and with it
    int bin;
    int cursor[kSearches];            // first CTA: tokens of each list
    uint32_t most[kMaxCluster], least[kMaxCluster], ties[kMaxCluster];  // of every CTA, in every CTA
    int nan[kMaxCluster];
    uint32_t block_most, block_least;
    int block_nan;
    int warp_counts[kWarps];
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_float(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) {
    return __bfloat162float(v);
}

template <typename T, bool CLUSTER>
class Row {
   public:
    __device__ Row(const SampleArgs &args, Shared &shared, unsigned char *dynamic) : a(args), sh(shared) {
        buf = reinterpret_cast<float *>(dynamic);
        lo = reinterpret_cast<uint32_t *>(buf + a.slots);
        hi = lo + kBins;
        scan = reinterpret_cast<u64 *>(hi + kBins);
        list = scan + kBins;
        list_own = list + kList;
        bitmap = reinterpret_cast<uint32_t *>(list_own + kList);
        tid = threadIdx.x;
        rank = CLUSTER ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
        ctas = CLUSTER ? static_cast<int>(cg::this_cluster().num_blocks()) : 1;
    }

    __device__ void run(int64_t row_index) {
        row = row_index;
        if (tid < kSearches) sh.cursor[tid] = 0;
        if (tid == 0) sh.block_most = 0, sh.block_least = 0xffffffffu, sh.block_nan = 0;
        clear_bins();
        load();
        share_extremes();
        settings();
        if (top == -INFINITY)
            finish(-1, 0, 1);
        else
            sample();
        sync_all();  // nobody leaves while another reads its shared memory
    }

   private:
    const SampleArgs &a;
    Shared &sh;
    float *buf;
    uint32_t *lo, *hi;  // histogram: 64-bit sums in two words
    u64 *scan, *list, *list_own;
    uint32_t *bitmap;
    int tid, rank, ctas, searches = 0;
    int64_t row;
    int start, count, phase, quads;  // first logit and number of this CTA's, offset of the first in buf, float4s of buf
    float top, lowest;               // largest and smallest logit above -inf
    float half_top, slices;          // slices of a unit of (top - v) / 2
    double wide_top, scale;
    int64_t top_k;
    float top_p, min_p, uniform;
    bool bad;
    bool limited = false;  // by top-k: tokens up to (limit_value, limit_index) in the order
    float limit_value;
    int limit_index;

    __device__ bool leader() const { return rank == 0; }
    __device__ void sync_all() {
        if (CLUSTER)
            cg::this_cluster().sync();
        else
            __syncthreads();
    }
    template <typename U>
    __device__ U *at(U *mine, int cta) const {
        return CLUSTER ? cg::this_cluster().map_shared_rank(mine, cta) : mine;
    }

    __device__ void clear_bins() {
        uint4 *words = reinterpret_cast<uint4 *>(lo);
        for (int i = tid; i < 2 * kBins / 4; i += kThreads) words[i] = make_uint4(0, 0, 0, 0);
    }

    // ---- the row -------------------------------------------------------------------------------------------
    // NaN as -inf (flagged), -0 as +0.
    __device__ float clean(float v, int &nan) {
        if (isnan(v)) {
            nan = 1;
            return -INFINITY;
        }
        return v + 0.0f;
    }

    __device__ void load() {
        constexpr int L = 16 / sizeof(T);
        start = rank * a.chunk;
        count = static_cast<int>(min(static_cast<int64_t>(a.chunk), a.vocab - start));
        const T *x = static_cast<const T *>(a.logits) + row * a.ld + start;
        phase = static_cast<int>(reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (L - 1);
        const int groups = (phase + count + L - 1) / L;  // of 16 bytes; the first and last may be parts
        quads = groups * L / 4;
        const bool ignores = a.ignore && (a.streams > 0 ? row % a.streams == 0 : row == 0);
        const bool edited = a.recent || ignores;
        if (a.recent)
            for (int i = tid; i < (count + 31) / 32; i += kThreads) bitmap[i] = 0;
        float most = -INFINITY, least = INFINITY;
        int nan = 0;
        auto note = [&](float v) {
            most = fmaxf(most, v);
            if (v > -INFINITY) least = fminf(least, v);
        };
        constexpr int kAhead = 4;
        for (int g0 = tid; g0 < groups; g0 += kAhead * kThreads) {
            uint4 raw[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int g = g0 + j * kThreads, e = g * L - phase;
                if (e >= 0 && e + L <= count) raw[j] = *reinterpret_cast<const uint4 *>(x + e);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int g = g0 + j * kThreads, e = g * L - phase;
                if (g >= groups) break;
                float v[L];
                if (e >= 0 && e + L <= count) {
                    const T *values = reinterpret_cast<const T *>(&raw[j]);
#pragma unroll
                    for (int i = 0; i < L; ++i) v[i] = to_float(values[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < L; ++i)
                        v[i] = e + i >= 0 && e + i < count ? to_float(x[e + i]) : -INFINITY;
                }
                if (!edited) {
#pragma unroll
                    for (int i = 0; i < L; ++i) {
                        v[i] = clean(v[i], nan);
                        note(v[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < L; i += 4)
                    *reinterpret_cast<float4 *>(buf + g * L + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            }
        }
        __syncthreads();
        if (edited) {
            float *const mine = buf + phase;
            if (a.recent)
                for (int64_t j = tid; j < a.recent_len; j += kThreads) {
                    const int64_t id = a.recent[row * a.recent_len + j], at_id = id - start;
                    if (id < 0 || id >= a.limit || at_id < 0 || at_id >= count) continue;
                    const uint32_t bit = 1u << (at_id & 31);
                    if (!(atomicOr(&bitmap[at_id >> 5], bit) & bit)) mine[at_id] = __fdiv_rn(mine[at_id], a.penalty);
                }
            __syncthreads();
            if (ignores)
                for (int64_t j = tid; j < a.n_ignore; j += kThreads) {
                    const int64_t at_id = a.ignore[j] - start;
                    if (at_id >= 0 && at_id < count) mine[at_id] = -INFINITY;
                }
            __syncthreads();
            for (int g = tid; g < quads; g += kThreads) {
                float4 &q = reinterpret_cast<float4 *>(buf)[g];
                q = make_float4(clean(q.x, nan), clean(q.y, nan), clean(q.z, nan), clean(q.w, nan));
                note(q.x), note(q.y), note(q.z), note(q.w);
            }
        }
        const uint32_t most_key = __reduce_max_sync(0xffffffffu, key_of(most));
        const uint32_t least_key = __reduce_min_sync(0xffffffffu, key_of(least));
        nan = __any_sync(0xffffffffu, nan);
        if ((tid & 31) == 0) {
            atomicMax(&sh.block_most, most_key);
            atomicMin(&sh.block_least, least_key);
            if (nan) sh.block_nan = 1;
        }
        __syncthreads();
    }

    // Largest and smallest key (and the NaN flag) of the row, from those of each CTA.
    __device__ void share_extremes() {
        if (CLUSTER) {
            if (tid < ctas) {
                *at(&sh.most[rank], tid) = sh.block_most;
                *at(&sh.least[rank], tid) = sh.block_least;
                *at(&sh.nan[rank], tid) = sh.block_nan;
            }
            sync_all();
        } else if (tid == 0) {
            sh.nan[0] = sh.block_nan;
        }
        uint32_t most = sh.block_most, least = sh.block_least;
        if (CLUSTER)
            for (int i = 0; i < ctas; ++i) most = max(most, sh.most[i]), least = min(least, sh.least[i]);
        top = value_of(most);
        lowest = value_of(least);
    }

    __device__ void settings() {
        bad = false;
        float temperature = a.temperature_rows ? a.temperature_rows[row] : a.temperature;
        if (!(temperature >= 0.0f) || isinf(temperature)) bad = true, temperature = 0.0f;
        top_k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
        if (top_k < 0) bad = true, top_k = 0;
        if (top_k == 0 || top_k > a.vocab) top_k = a.vocab;
        top_p = a.top_p_rows ? a.top_p_rows[row] : a.top_p;
        if (!(top_p >= 0.0f && top_p <= 1.0f)) bad = true, top_p = top_p < 0.0f ? 0.0f : 1.0f;
        min_p = a.min_p_rows ? a.min_p_rows[row] : a.min_p;
        if (!(min_p >= 0.0f && min_p <= 1.0f)) bad = true, min_p = min_p > 1.0f ? 1.0f : 0.0f;
        uniform = a.uniforms[row];
        if (!(uniform >= 0.0f && uniform < 1.0f)) bad = true, uniform = uniform >= 1.0f ? 1.0f : 0.0f;
        if (temperature == 0.0f) top_k = 1;
        scale = temperature > 0.0f ? 1.4426950408889634074 / static_cast<double>(temperature) : 0.0;
        if (top == INFINITY) {  // +inf alone has weight: as 0 among -inf
            for (int g = tid; g < quads; g += kThreads) {
                float4 &q = reinterpret_cast<float4 *>(buf)[g];
                q.x = q.x == top ? 0.0f : -INFINITY, q.y = q.y == top ? 0.0f : -INFINITY;
                q.z = q.z == top ? 0.0f : -INFINITY, q.w = q.w == top ? 0.0f : -INFINITY;
            }
            top = lowest = 0.0f;
            __syncthreads();
        }
        // Half differences, so that none overflows.  The slices reach to the lowest logit, or to 31.9 T below the top,
        // where weights are below 2^-45 and round to nothing.
        half_top = 0.5f * top;
        wide_top = top;
        const float reach = fminf(__fmaf_rn(-0.5f, lowest, half_top), 15.95f * temperature);
        slices = fminf(__fdiv_rn(static_cast<float>(kBins - 1), reach), FLT_MAX);
    }

    // Slice of a logit: never smaller for a smaller logit; kBins and above where there is no weight (-inf among it).
    // The sum with 2^23 leaves the nearest integer in the low bits.
    __device__ uint32_t bin_of(float v) const {
        const float d = __fmaf_rn(-0.5f, v, half_top);
        return __float_as_uint(__fmaf_rn(d, slices, 8388608.0f)) - 0x4b000000u;
    }
    __device__ bool within(float v, int index) const {
        return v > limit_value || (v == limit_value && index <= limit_index);
    }
    __device__ u64 weight(float v) const { return weight_of(v, wide_top, scale); }

    // f(logits, slices, index of the first) for this CTA's tokens by fours; a token without weight, or beyond the
    // limit of top-k, has a slice of kBins or above.
    template <typename F>
    __device__ void for_fours(F f) {
        for (int g = tid; g < quads; g += kThreads) {
            const float4 q = reinterpret_cast<const float4 *>(buf)[g];
            const float v[4] = {q.x, q.y, q.z, q.w};
            const int first = start + 4 * g - phase;
            uint32_t bin[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) bin[i] = bin_of(v[i]);
            if (limited) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!within(v[i], first + i)) bin[i] = kBins;
            }
            f(v, bin, first);
        }
    }

    // ---- histograms ----------------------------------------------------------------------------------------
    __device__ void add(uint32_t bin, u64 w) {
        const uint32_t low = static_cast<uint32_t>(w);
        const uint32_t old = atomicAdd(&lo[bin], low);
        const uint32_t high = static_cast<uint32_t>(w >> 32) + (old + low < old);
        if (high) atomicAdd(&hi[bin], high);
    }

    // Running sums of the cluster's histogram, in the first CTA: scan[bin] = what lies before it.
    __device__ void running_sums() {
        sync_all();
        if (CLUSTER) {
            const int share = kBins / ctas;
            for (int i = tid; i < share; i += kThreads) {
                const int bin = rank * share + i;
                u64 sum = 0;
                for (int c = 0; c < ctas; ++c)
                    sum += (static_cast<u64>(*at(&hi[bin], c)) << 32) + *at(&lo[bin], c);
                *at(&scan[bin], 0) = sum;
            }
            sync_all();
        }
        if (!leader()) return;
        constexpr int kEach = kBins / kThreads;
        u64 own[kEach], sum = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int bin = tid * kEach + i;
            own[i] = CLUSTER ? scan[bin] : (static_cast<u64>(hi[bin]) << 32) + lo[bin];
            sum += own[i];
        }
        u64 all;
        u64 before = sum_before(sum, all);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            scan[tid * kEach + i] = before;
            before += own[i];
        }
        if (tid == 0) sh.total = all;
        __syncthreads();
    }

    // The slice that `target` (below the total; the first CTA's) falls into, told to every CTA.
    __device__ void locate(u64 target) {
        if (leader()) {
            constexpr int kEach = kBins / kThreads;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int bin = tid * kEach + i;
                const u64 next = bin + 1 < kBins ? scan[bin + 1] : sh.total;
                if (scan[bin] <= target && target < next)
                    for (int c = 0; c < ctas; ++c) {
                        Shared &to = *at(&sh, c);
                        to.bin = bin;
                        to.before = scan[bin];
                        to.upto = next;
                        to.target = target;
                    }
            }
        }
        sync_all();
    }

    // Collects the tokens whose slice lies in [from, to] and whose key in [low, high] in the first CTA's list; returns
    // how many there are (kList are held).
    __device__ int collect(uint32_t from, uint32_t to, uint32_t low = 0, uint32_t high = 0xffffffffu) {
        int *const cursor = at(&sh.cursor[searches], 0);
        u64 *const into = at(list, 0);
        for_fours([&](const float(&v)[4], const uint32_t(&bin)[4], int first) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) any |= bin[i] - from <= to - from;
            if (!any) return;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t key = key_of(v[i]);
                if (bin[i] - from > to - from || key < low || key > high) continue;
                const int place = atomicAdd(cursor, 1);
                if (place < kList) into[place] = order_of(v[i], first + i);
            }
        });
        sync_all();
        ++searches;
        return *cursor;
    }

    // First CTA: the n listed tokens in order, one a thread (all ones behind them).  A bitonic network: strides below a
    // warp by shuffles, the others through two arrays in turn.
    __device__ u64 sorted(int n) {
        u64 mine = tid < n ? list[tid] : ~0ull;
        u64 *area = list_own, *next = list;
        __syncthreads();
        for (int size = 2; size < 2 * n; size <<= 1)
            for (int stride = size >> 1; stride > 0; stride >>= 1) {
                u64 other;
                if (stride >= 32) {
                    area[tid] = mine;
                    __syncthreads();
                    other = area[tid ^ stride];
                    u64 *const t = area;
                    area = next;
                    next = t;
                } else {
                    other = __shfl_xor_sync(0xffffffffu, mine, stride);
                }
                const bool smaller = ((tid & stride) == 0) == ((tid & size) == 0);
                if ((other < mine) == smaller) mine = other;
            }
        __syncthreads();
        return mine;
    }

    // Running sum over the CTA's threads (what lies before this one); `all`: the whole.
    __device__ u64 sum_before(u64 own, u64 &all) {
        u64 upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, upto, o);
            if ((tid & 31) >= o) upto += v;
        }
        if ((tid & 31) == 31) sh.warp_sums[tid >> 5] = upto;
        __syncthreads();
        u64 before = upto - own;
        all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w == (tid >> 5)) before += all;
            all += sh.warp_sums[w];
        }
        __syncthreads();
        return before;
    }

    static __device__ float value_in(u64 order) { return value_of(~static_cast<uint32_t>(order >> 32)); }
    static __device__ int index_in(u64 order) { return static_cast<int>(static_cast<uint32_t>(order)); }

    // First CTA: which of the n listed tokens the target falls into.
    __device__ void rank_list(int n, u64 before, u64 target, bool by_weight) {
        const u64 mine = sorted(n);
        const u64 own = tid >= n ? 0 : by_weight ? weight(value_in(mine)) : 1;
        u64 all;
        const u64 sum = before + sum_before(own, all);
        if (sum <= target && target < sum + own) sh.found = {mine, sum, own};
        __syncthreads();
    }

    // The token of the located slice that the target falls into: in the first CTA's sh.found.  A slice with too many
    // tokens costs the histogram (returns false then).
    __device__ bool search_slice(bool by_weight) {
        const uint32_t slice = sh.bin;
        u64 before = sh.before;
        const u64 target = sh.target;
        int n = collect(slice, slice);
        if (n <= kList) {
            if (leader()) rank_list(n, before, target, by_weight);
            return true;
        }
        uint32_t low_key = 0, high_key = 0xffffffffu;
        for (;;) {
            auto member = [&](float v, uint32_t bin) {
                const uint32_t key = key_of(v);
                return bin == slice && key >= low_key && key <= high_key;
            };
            // keys of the slice that is left
            uint32_t most = 0, least = 0xffffffffu, group = 0;
            if (tid == 0) sh.block_most = 0, sh.block_least = 0xffffffffu;
            clear_bins();
            __syncthreads();
            for_fours([&](const float(&v)[4], const uint32_t(&bin)[4], int) {
                for (int i = 0; i < 4; ++i)
                    if (member(v[i], bin[i])) {
                        most = max(most, key_of(v[i])), least = min(least, key_of(v[i]));
                        ++group;
                    }
            });
            most = __reduce_max_sync(0xffffffffu, most);
            least = __reduce_min_sync(0xffffffffu, least);
            group = __reduce_add_sync(0xffffffffu, group);
            if ((tid & 31) == 0) {
                atomicMax(&sh.block_most, most);
                atomicMin(&sh.block_least, least);
                sh.warp_counts[tid >> 5] = static_cast<int>(group);
            }
            __syncthreads();
            if (tid < ctas) {
                uint32_t all = 0;
                for (int w = 0; w < kWarps; ++w) all += sh.warp_counts[w];
                Shared &to = *at(&sh, tid);
                to.most[rank] = sh.block_most;
                to.least[rank] = sh.block_least;
                to.ties[rank] = all;
            }
            sync_all();
            most = 0, least = 0xffffffffu;
            for (int i = 0; i < ctas; ++i) most = max(most, sh.most[i]), least = min(least, sh.least[i]);
            if (most == least) {
                const u64 own = by_weight ? weight(value_of(most)) : 1;
                u64 place = (target - before) / own;
                u64 skipped = 0;
                int holder = 0;
                while (holder + 1 < ctas && place - skipped >= sh.ties[holder]) skipped += sh.ties[holder++];
                const int index = holder == rank ? nth(value_of(most), static_cast<uint32_t>(place - skipped)) : 0;
                if (holder == rank && index >= 0)
                    at(&sh, 0)->found = {order_of(value_of(most), index), before + place * own, own};
                sync_all();
                return false;
            }
            int shift = 0;
            while (((most - least) >> shift) >= kBins) ++shift;
            for_fours([&](const float(&v)[4], const uint32_t(&bin)[4], int) {
                for (int i = 0; i < 4; ++i)
                    if (member(v[i], bin[i])) add((most - key_of(v[i])) >> shift, by_weight ? weight(v[i]) : 1);
            });
            running_sums();
            locate(target - before);
            before += sh.before;
            high_key = most - (static_cast<uint32_t>(sh.bin) << shift);
            low_key = max(least, high_key - ((1u << shift) - 1));
            n = collect(slice, slice, low_key, high_key);
            if (n <= kList) {
                if (leader()) rank_list(n, before, target, by_weight);
                return false;
            }
        }
    }

    // Index of this CTA's n-th (from 0) token with that logit: in the thread that holds it, -1 in the others.
    __device__ int nth(float value, uint32_t n) {
        uint32_t before = 0;
        int found = -1;
        for (int i0 = 0; i0 < count && before <= n; i0 += kThreads) {
            const int i = i0 + tid;
            const bool is = i < count && buf[phase + i] == value;
            const uint32_t vote = __ballot_sync(0xffffffffu, is);
            __syncthreads();
            if ((tid & 31) == 0) sh.warp_counts[tid >> 5] = __popc(vote);
            __syncthreads();
            uint32_t mine = before + __popc(vote & ((1u << (tid & 31)) - 1));
            for (int w = 0; w < kWarps; ++w) {
                if (w < (tid >> 5)) mine += sh.warp_counts[w];
                before += sh.warp_counts[w];
            }
            if (is && mine == n) found = start + i;
        }
        return found;
    }

    // ---- the filters and the draw ----------------------------------------------------------------------------
    __device__ u64 least_weight() const {
        return static_cast<u64>(ceil(static_cast<double>(min_p) * 17592186044416.0));  // 2^44
    }

    // The histogram of weights and its running sums; what min-p leaves of them to the first CTA.
    __device__ void weigh() {
        const u64 least = least_weight();
        u64 passing = 0;
        for_fours([&](const float(&v)[4], const uint32_t(&bin)[4], int) {
            if (bin[0] >= kBins && bin[1] >= kBins && bin[2] >= kBins && bin[3] >= kBins) return;
            u64 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = weight(bin[i] < kBins ? v[i] : top);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (bin[i] < kBins) {
                    add(bin[i], w[i]);
                    if (w[i] >= least) passing += w[i];
                }
        });
        if (min_p > 0.0f) {
            u64 all;
            sum_before(passing, all);
            if (tid == 0) at(&sh, 0)->passing[rank] = all;
        }
        running_sums();
    }

    // Weight that is kept of `all`: up to the token that passes top-p, and no more than min-p lets pass.
    __device__ u64 drawn(u64 kept) const {
        const u64 place = static_cast<u64>(static_cast<double>(uniform) * static_cast<double>(kept));
        return min(place, kept - 1);
    }
    __device__ u64 nucleus(u64 all) const {  // the weight whose token is the last that top-p keeps
        const u64 part = static_cast<u64>(ceil(static_cast<double>(top_p) * static_cast<double>(all)));
        return max(part, u64(1)) - 1;
    }

    // First CTA: all that can be drawn is in the list (n tokens and no more): filters and draw over it in order.
    __device__ void sample_list(int n) {
        const u64 mine = sorted(n);
        const u64 own = tid < min(static_cast<int64_t>(n), top_k) ? weight(value_in(mine)) : 0;
        u64 kept, passing;
        const u64 before = sum_before(own, kept);
        if (top_p < 1.0f) {
            const u64 target = nucleus(kept);
            if (before <= target && target < before + own) sh.total = before + own;
            __syncthreads();
            kept = sh.total;
        }
        if (min_p > 0.0f) {
            sum_before(own >= least_weight() ? own : 0, passing);
            kept = min(kept, passing);
        }
        const u64 target = drawn(kept);
        if (before <= target && target < before + own) sh.found = {mine, before, own};
        __syncthreads();
        finish(index_in(sh.found.order), sh.found.own, kept);
    }

    __device__ void sample() {
        if (a.vocab <= kList) {
            const int n = collect(0, kBins - 1);
            if (leader()) sample_list(n);
            return;
        }
        if (top_k < a.vocab) {
            for_fours([&](const float(&)[4], const uint32_t(&bin)[4], int) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (bin[i] < kBins) atomicAdd(&lo[bin[i]], 1u);
            });
            running_sums();
            locate(leader() ? min(static_cast<u64>(top_k), sh.total) - 1 : 0);
            // The k-th token's slice, or the last one with a token.  Few enough up to it: the first CTA has them all.
            if (sh.upto <= kList) {
                const int n = collect(0, sh.bin);
                if (leader()) sample_list(n);
                return;
            }
            if (sh.target + 1 == static_cast<u64>(top_k)) {
                search_slice(false);
                if (CLUSTER) {
                    if (leader() && tid > 0 && tid < ctas) at(&sh, tid)->found = sh.found;
                    sync_all();
                }
                limited = true;
                limit_value = value_in(sh.found.order);
                limit_index = index_in(sh.found.order);
            }
            sync_all();  // the histograms have been read
            clear_bins();
            __syncthreads();
        }
        weigh();
        u64 kept = leader() ? sh.total : 0;
        if (top_p < 1.0f) {
            locate(leader() ? nucleus(kept) : 0);
            const bool whole = search_slice(true);
            kept = leader() ? sh.found.before + sh.found.own : 0;
            if (!whole) {
                sync_all();
                clear_bins();
                __syncthreads();
                weigh();
            }
        }
        if (min_p > 0.0f && leader()) {
            u64 passing = 0;
            for (int c = 0; c < ctas; ++c) passing += sh.passing[c];
            kept = min(kept, passing);
        }
        locate(leader() ? drawn(kept) : 0);
        search_slice(true);
        finish(index_in(sh.found.order), sh.found.own, kept);
    }

    __device__ void finish(int token, u64 own, u64 kept) {
        if (!leader() || tid != 0) return;
        a.out[row] = max(token, 0);
        if (a.logprob)
            a.logprob[row] = token < 0 ? -INFINITY
                                       : static_cast<float>(log(static_cast<double>(own) / static_cast<double>(kept)));
        int flags = (token < 0 ? LEVO_SAMPLE_EMPTY : 0) | (bad ? LEVO_SAMPLE_PARAM : 0);
        for (int c = 0; c < ctas; ++c) flags |= sh.nan[c] ? LEVO_SAMPLE_NAN : 0;
        if (a.status && flags) atomicOr(a.status, flags);
    }
};

template <typename T, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ Shared shared;
    Row<T, CLUSTER> row(a, shared, dynamic);
    row.run(CLUSTER ? blockIdx.x / cg::this_cluster().num_blocks() : blockIdx.x);
}

template <typename T>
int launch_sample(SampleArgs &a, const char *what, cudaStream_t stream) {
    constexpr int L = 16 / sizeof(T);
    auto chunk_of = [&](int ctas) { return static_cast<int>((a.vocab + ctas - 1) / ctas + 7) / 8 * 8; };
    auto smem_of = [&](int ctas) {
        const size_t slots = (chunk_of(ctas) + 2 * L + 3) / 4 * 4, words = a.recent ? (chunk_of(ctas) + 31) / 32 : 0;
        return slots * sizeof(float) + 2 * kBins * sizeof(uint32_t) + (kBins + 2 * kList) * sizeof(u64) + words * 4;
    };
    // As many CTAs a row as leave every CTA work, while the SMs (two CTAs each) are not filled by the rows.
    int ctas = 1;
    while (ctas < kMaxCluster && (smem_of(ctas) > 110 * 1024 ||
                                  (a.rows * ctas * 2 <= 2LL * sm_count() && a.vocab / ctas >= 4096)))
        ctas *= 2;
    a.chunk = chunk_of(ctas);
    a.slots = (a.chunk + 2 * L + 3) / 4 * 4;
    if (a.rows * ctas > 0x7fffffff)
        return set_error(LEVO_OPS_EUNSUPPORTED, std::string(what) + ": too many rows for one call");
    // Above 48 KB with the static part the kernel has to opt in, which resident_ctas does from the dynamic part alone.
    size_t smem = smem_of(ctas);
    if (smem + sizeof(Shared) > 48 * 1024) smem = std::max<size_t>(smem, 48 * 1024 + 16);
    const void *kernel = ctas > 1 ? reinterpret_cast<const void *>(sample_kernel<T, true>)
                                  : reinterpret_cast<const void *>(sample_kernel<T, false>);
    int per_sm = 0;
    if (resident_ctas(kernel, kThreads, smem, &per_sm) != cudaSuccess) return check_launch(what);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows * ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 1 : 0;
    const cudaError_t err = ctas > 1 ? cudaLaunchKernelEx(&cfg, sample_kernel<T, true>, a)
                                     : cudaLaunchKernelEx(&cfg, sample_kernel<T, false>, a);
    (void)err;
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
    SampleArgs a{s.logits, s.rows, s.vocab, s.ld, s.uniforms, s.temperature_rows, s.top_p_rows, s.min_p_rows,
                       s.top_k_rows, s.temperature, s.top_p, s.min_p, s.penalty, s.top_k,
                       s.recent_len > 0 ? s.recent : nullptr, s.recent_len, limit,
                       s.n_ignore > 0 ? s.ignore : nullptr, s.n_ignore, s.streams, s.tokens_out, s.logprob_out,
                       s.status, 0, 0};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (s.dtype == LEVO_DTYPE_F32) return launch_sample<float>(a, w, st);
    if (s.dtype == LEVO_DTYPE_F16) return launch_sample<__half>(a, w, st);
    return launch_sample<__nv_bfloat16>(a, w, st);
}

}  // extern "C"
