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

__device__ __forceinline__ u64 weight_of(float v, float top, double scale) {
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
    u64 before;                       // of the slice that the target falls into
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
        if (top == -INFINITY) {
            if (leader()) finish(-1, 0, 1);
        } else {
            sample();
        }
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
    float half_top, reach, slices;   // (top - v) / 2 up to `reach` has weight; slices of it a unit
    double scale;
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
        // Half differences, so that none overflows.  31.9 T and more below the maximum there is no weight (2^-46).
        half_top = 0.5f * top;
        reach = isinf(top) ? 0.0f : fminf(__fmaf_rn(-0.5f, lowest, half_top), 15.95f * temperature);
        slices = fminf(__fdiv_rn(static_cast<float>(kBins), reach), FLT_MAX);
    }

    // Slice of a logit (never larger for a larger logit), or -1 where it has no weight.
    __device__ int bin_of(float v) const {
        const float d = v == top ? 0.0f : __fmaf_rn(-0.5f, v, half_top);
        if (!(d <= reach)) return -1;
        return min(kBins - 1, static_cast<int>(d * slices));
    }
    __device__ bool within(float v, int index) const {
        return !limited || v > limit_value || (v == limit_value && index <= limit_index);
    }
    __device__ u64 weight(float v) const { return weight_of(v, top, scale); }

    // f(logit, index, slice) for every token of this CTA that has weight and that top-k has left.
    template <typename F>
    __device__ void for_each(F f) {
        for (int g = tid; g < quads; g += kThreads) {
            const float4 q = reinterpret_cast<const float4 *>(buf)[g];
            const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int bin = bin_of(v[i]), index = start + 4 * g + i - phase;
                if (bin >= 0 && within(v[i], index)) f(v[i], index, bin);
            }
        }
    }

    // ---- histograms ----------------------------------------------------------------------------------------
    __device__ void add(int bin, u64 w) {
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
        u64 upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, upto, o);
            if ((tid & 31) >= o) upto += v;
        }
        if ((tid & 31) == 31) sh.warp_sums[tid >> 5] = upto;
        __syncthreads();
        u64 before = upto - sum, all = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w == (tid >> 5)) before += all;
            all += sh.warp_sums[w];
        }
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
                        to.target = target;
                    }
            }
        }
        sync_all();
    }

    // Collects the tokens that `member` takes in the first CTA's list; returns how many there are (kList are held).
    template <typename M>
    __device__ int collect(M member) {
        int *const cursor = at(&sh.cursor[searches], 0);
        u64 *const to = at(list, 0);
        for_each([&](float v, int index, int bin) {
            if (!member(v, bin)) return;
            const int place = atomicAdd(cursor, 1);
            if (place < kList) to[place] = order_of(v, index);
        });
        sync_all();
        ++searches;
        return *cursor;
    }

    // First CTA: which of the n listed tokens the target falls into.  Several threads a token add up the list.
    __device__ void rank_list(int n, u64 before, u64 target, bool by_weight) {
        for (int i = tid; i < n; i += kThreads)
            list_own[i] = by_weight ? weight(value_of(~static_cast<uint32_t>(list[i] >> 32))) : 1;
        __syncthreads();
        int share = 32;
        while (share > 1 && n * share > kThreads) share >>= 1;
        const int lane = tid % share;
        for (int i = tid / share; i - tid / share < n; i += kThreads / share) {
            const u64 mine = i < n ? list[i] : 0;
            u64 sum = 0;
            for (int j = lane; j < n; j += share)
                if (list[j] < mine) sum += list_own[j];
            for (int o = share / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0 && i < n && before + sum <= target && target < before + sum + list_own[i])
                sh.found = {mine, before + sum, list_own[i]};
        }
        __syncthreads();
    }

    // The token that `target` falls into: in the first CTA's sh.found.  running_sums() went before; a slice with too
    // many tokens costs the histogram (returns false then).
    __device__ bool search(u64 target, bool by_weight) {
        locate(target);
        const int bin = sh.bin;
        u64 before = sh.before;
        target = sh.target;
        int n = collect([&](float, int b) { return b == bin; });
        if (n <= kList) {
            if (leader()) rank_list(n, before, target, by_weight);
            return true;
        }
        uint32_t low_key = 0, high_key = 0xffffffffu;
        for (;;) {
            auto member = [&](float v, int b) {
                const uint32_t key = key_of(v);
                return b == bin && key >= low_key && key <= high_key;
            };
            // keys of the slice that is left
            uint32_t most = 0, least = 0xffffffffu, group = 0;
            if (tid == 0) sh.block_most = 0, sh.block_least = 0xffffffffu;
            clear_bins();
            __syncthreads();
            for_each([&](float v, int, int b) {
                if (!member(v, b)) return;
                most = max(most, key_of(v)), least = min(least, key_of(v));
                ++group;
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
            for_each([&](float v, int, int b) {
                if (member(v, b)) add(static_cast<int>((most - key_of(v)) >> shift), by_weight ? weight(v) : 1);
            });
            running_sums();
            locate(target - before);
            before += sh.before;
            high_key = most - (static_cast<uint32_t>(sh.bin) << shift);
            low_key = max(least, high_key - ((1u << shift) - 1));
            n = collect(member);
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
    __device__ void weigh() {
        const u64 least = static_cast<u64>(ceil(static_cast<double>(min_p) * 17592186044416.0));  // 2^44
        u64 passing = 0;
        for_each([&](float v, int, int bin) {
            const u64 w = weight(v);
            add(bin, w);
            if (w >= least) passing += w;
        });
        if (min_p > 0.0f) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) passing += __shfl_xor_sync(0xffffffffu, passing, o);
            __syncthreads();
            if ((tid & 31) == 0) sh.warp_sums[tid >> 5] = passing;
            __syncthreads();
            if (tid == 0) {
                u64 all = 0;
                for (int w = 0; w < kWarps; ++w) all += sh.warp_sums[w];
                at(&sh, 0)->passing[rank] = all;
            }
        }
        running_sums();
    }

    __device__ void sample() {
        if (top_k < a.vocab) {
            for_each([&](float, int, int bin) { atomicAdd(&lo[bin], 1u); });
            running_sums();
            sync_all();  // every CTA asks for the total of the first
            const bool cuts = *at(&sh.total, 0) > static_cast<u64>(top_k);
            if (cuts) {
                search(static_cast<u64>(top_k) - 1, false);
                if (CLUSTER) {
                    if (leader() && tid > 0 && tid < ctas) at(&sh, tid)->found = sh.found;
                    sync_all();
                }
                limited = true;
                limit_value = value_of(~static_cast<uint32_t>(sh.found.order >> 32));
                limit_index = static_cast<int>(static_cast<uint32_t>(sh.found.order));
                if (top_k == 1) {
                    if (leader()) finish(limit_index, 1, 1);
                    return;
                }
            }
            __syncthreads();
            if (CLUSTER) sync_all();  // the histograms have been read
            clear_bins();
            __syncthreads();
        }
        weigh();
        u64 kept = leader() ? sh.total : 0;
        if (top_p < 1.0f) {
            const double part = ceil(static_cast<double>(top_p) * static_cast<double>(kept));
            const u64 target = leader() ? max(1ull, static_cast<u64>(part)) - 1 : 0;
            const bool whole = search(target, true);
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
        const u64 target =
            leader() ? min(static_cast<u64>(static_cast<double>(uniform) * static_cast<double>(kept)), kept - 1) : 0;
        search(target, true);
        if (leader()) finish(static_cast<int>(static_cast<uint32_t>(sh.found.order)), sh.found.own, kept);
    }

    __device__ void finish(int token, u64 own, u64 kept) {
        if (tid != 0) return;
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
