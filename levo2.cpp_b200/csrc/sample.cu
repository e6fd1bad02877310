// Next-token sampling from one given uniform number a row: temperature, top-k,
// top-p and min-p over logits that the penalty and the ignore list of the greedy
// selection have gone through (the formulas stand at levo_sampling).
//
// All three filters keep a prefix of one order (larger logit first, equal logits
// by index), and the draw is a place in that prefix.  So the row is not sorted:
// top-k, top-p and the draw are each the search for the one token at which a
// running count, or a running weight, passes a target:
//   1. a histogram (of counts, or of weights) over equal slices of the logits'
//      range below the maximum, and its running sums;
//   2. the slice that the target falls into;
//   3. its tokens, some tens of 16385, in a list; each adds up what lies before it.
// A slice of more than kList tokens (many equal or close logits) is cut further by
// the bits of its keys until its tokens are few or all equal.  Two shortcuts:
//   - top-k up to kList: the k-th largest of the threads' own largest logits is a
//     lower bound of the k-th largest, and few tokens lie between (k = 50 of 16385
//     over 512 threads: about 53 in all).  They are listed and ordered, and the
//     rest happens in the list;
//   - top-p and the draw: what top-p keeps is known to a slice before its token is
//     found, which mostly fixes the draw's slice as well: one pass lists both.
//
// Weights are F64 exponentials rounded to multiples of 2^-44 of the largest and
// summed as 64-bit integers (131072 * 2^44 = 2^61): exact, in any order, so that
// atomics and the split over CTAs cannot change a result.  F32 sums would put one
// flat row in some hundreds on another token: a border lies within 1e-7 of one of
// 1e5 others.
//
// A CTA's share of a row is held in shared memory as F32 and read from HBM once; a
// share that does not fit (beside a second CTA, where there are many) is read again
// from L2, by a ring of cp.async copies.  Rows that are few and long are split over a cluster,
// whose first CTA merges the histograms, takes the decisions and holds the lists.
//
// What bounds it: instruction issue, not bytes.  1024 rows of 16385 in F16 (six in ten
// over the whole vocabulary) take 72 us, 5.1 us of HBM time: 44 million warp
// instructions in 62 % of the issue slots, 84 a logit on the average of all rows.
// 128 flat F32 rows of 131072, where every logit is weighed (11 F64 operations each),
// take 101 us: 107 a logit in 59 % of the slots.  Small batches are bound by the
// chain of some ten phases between barriers, 1 to 2 us each for a cluster.
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
static_assert(kWarps <= 32 && (kWarps & (kWarps - 1)) == 0, "a warp's lanes read all warps' values");
constexpr int kBins = 4096;      // slices of a histogram of weights
constexpr int kCountBins = 512;  // and of one of counts
constexpr int kList = 512;
static_assert(kList == kThreads, "a listed token a thread");
constexpr int kMaxCluster = 8;
constexpr int kOneShare = 32768;  // logits that a row is split from
constexpr int kMostHeld = 32768;  // that a CTA holds: a bit each in a thread's 64
// Groups that a thread has on their way when it reads a row again.  Four leave room for a second CTA on the SM beside
// the bits of 131072 edited ids; eight did not, and 128 rows of 131072 with a penalty took 153 us instead of 117 (300 of
// 20011 72 and 56); without one the two differ by 3 % (104 and 101; 48 and 47).
constexpr int kRing = 4;
// Slices are at least 2^-128 of (top - v) / 2 wide, so from 15.95 T = 2^-116 down kBins of them end beyond the weights.
constexpr float kTinyTemperature = 1e-36f;
constexpr int kSearches = 24;  // lists of one row: three searches with up to four further cuts each, and three more
constexpr int64_t kMaxVocab = int64_t(1) << 17;
constexpr int kHalfAnSm = 112 * 1024;  // shared memory of a CTA that leaves room for a second one

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
    int chunk, slots, words;  // logits of a CTA, their places and the words of their bits in shared memory
};

// Integers in the order of the values (-0 is made +0).
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
// The order as one integer, ascending: larger logit first, then the smaller index.
__device__ __forceinline__ u64 order_of(float v, int index) {
    return (static_cast<u64>(~key_of(v)) << 32) | static_cast<uint32_t>(index);
}

// exp((v - top) / T) in units of 2^-44.  y = (v - top) * 64 log2(e)/T in F64, k the
// nearest integer, g = y - k: 2^(44 + k/64), from a table of 2^(44 + j/64), times the
// Taylor series of 2^(g/64), |g| <= 1/2, to degree 4 (the first term left out is
// (ln2/128)^5 / 5! = 3.9e-14, below the unit).
constexpr int kSteps = 64;
constexpr double kLn2 = 0.693147180559945309417;
constexpr double step_coefficient(int k) {  // of g^k
    double c = 1.0;
    for (int i = 1; i <= k; ++i) c *= kLn2 / kSteps / i;
    return c;
}

// 2^(44 + j/64): the Taylor series of 2^f, |f| <= 1/2, to degree 18, as the compiler evaluates it.
struct StepPowers {
    double v[kSteps];
    constexpr StepPowers() : v() {
        for (int j = 0; j < kSteps; ++j) {
            const double x = kLn2 * (j < kSteps / 2 ? j : j - kSteps) / kSteps;
            double p = 1.0;
            for (int k = 18; k > 0; --k) p = 1.0 + p * x / k;
            v[j] = p * (j < kSteps / 2 ? 17592186044416.0 : 35184372088832.0);
        }
    }
};
__device__ const StepPowers kStepPowers{};

// For v within 32 T of the top, as bin_of and `seen` take them: the result is below 2^45 and its exponent above -3.
__device__ __forceinline__ u64 weight_of(float v, double top, double scale, const double *powers) {
    const double y = (static_cast<double>(v) - top) * scale;
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
    const double r = y + kRound;
    const int k = __double2loint(r);
    const double g = y - (r - kRound);
    double p = __fma_rn(step_coefficient(4), g, step_coefficient(3));
    p = __fma_rn(p, g, step_coefficient(2));
    p = __fma_rn(p, g, step_coefficient(1)) * g;
    const double power = powers[k & (kSteps - 1)];
    const double t = __hiloint2double(__double2hiint(power) + ((k & -kSteps) << 14), __double2loint(power));
    // adding 2^52 rounds to an integer in the low mantissa bits
    const double w = __fma_rn(t, p, t) + 4503599627370496.0;
    return static_cast<u64>(__double_as_longlong(w)) & ((1ull << 52) - 1);
}

// A slice of the histogram: what lies before it, and with it.
struct Slice {
    int bin;
    u64 before, upto;
};

// A row's settings, with the values out of range replaced.
struct Settings {
    int64_t top_k;
    float temperature, top_p, min_p, uniform;
    int bad;
};

// Largest and smallest key, and whether there is a NaN.
struct Extremes {
    uint32_t most, least;
    int nan;
};

// A token found: its place in the order, what lies before it, and what it has itself (weight, or 1).
struct Found {
    u64 order, before, own;
};

struct Shared {
    double powers[kSteps];
    u64 warp_sums[kWarps];            // of a running sum; at first each warp's largest and smallest key
    u64 total;                        // first CTA: of the histogram
    u64 passing[kMaxCluster];         // first CTA: weight that min-p leaves, of each CTA
    Found found;
    u64 target;
    int place;                        // of this CTA's first token in the list
    Slice slice, other;               // the one that the target falls into; the draw's, where it is known with top-p's
    int joint;                        // it is
    Settings set;
    int cursor[kSearches];            // first CTA: tokens of each list
    Extremes own;                     // of this CTA's share
    int nan;                          // the row has a NaN
    uint32_t most[kMaxCluster], least[kMaxCluster], ties[kMaxCluster];  // of every CTA, in every CTA
    uint32_t block_most, block_least;
    int warp_counts[kWarps];          // at first whether a warp has met a NaN
    int places[kThreads], ends[kThreads];  // of a list's slices
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

// 16-byte groups whose loads a thread has on their way when it reads a row that is held.  Two, four and nine of them,
// in us from L2 (from HBM): 192 F32 rows of 16385 15.5, 15.0, 16.2 (17.4, 17.4, 20.0), 60 of 32000 24.0, 22.9, 23.5
// (27.8, 24.9, 24.5), 192 of 8000 10.2, 10.0, 10.6; for the 16-bit types two and four: 60 rows of 32000 27.8, 27.3
// (30.0, 30.1), 192 of 16385 11.7, 11.7 (12.7, 13.0).
constexpr int kAhead = 4;

template <typename T, bool CLUSTER, bool HELD>
class Row {
   public:
    __device__ Row(const SampleArgs &args, Shared &shared) : a(args), sh(shared) {
        tid = threadIdx.x;
        rank = CLUSTER ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
        ctas = CLUSTER ? static_cast<int>(cg::this_cluster().num_blocks()) : 1;
    }

    __device__ __forceinline__ void run(int64_t row_index) {
        row = row_index;
        if (tid < kSearches) sh.cursor[tid] = 0;
        if (tid < kSteps) sh.powers[tid] = kStepPowers.v[tid];
        ask();
        load();
        share_extremes();
        settings();
        if (top == -INFINITY) {
            if (leader() && tid == 0) {
                a.out[row] = 0;
                if (a.logprob) a.logprob[row] = -INFINITY;
                flag(LEVO_SAMPLE_EMPTY);
            }
        } else {
            sample();
        }
        sync_all();  // nobody leaves while another reads its shared memory
    }

   private:
    const SampleArgs &a;
    Shared &sh;
    // The dynamic shared memory, at offsets that the compiler knows (pointers to it would hold registers).
    static __device__ __forceinline__ unsigned char *dynamic(size_t offset) {
        extern __shared__ __align__(16) unsigned char memory[];
        return memory + offset;
    }
    // Histogram, then its running sums (first CTA): 64 bits in two words.
    static __device__ __forceinline__ uint32_t *lo() { return reinterpret_cast<uint32_t *>(dynamic(0)); }
    static __device__ __forceinline__ uint32_t *hi() { return lo() + kBins; }
    static __device__ __forceinline__ u64 *list() { return reinterpret_cast<u64 *>(hi() + kBins); }
    static __device__ __forceinline__ u64 *spare() { return list() + kList; }
    // HELD: this CTA's logits, as the order sees them.  Else: groups on their way.
    static __device__ __forceinline__ float *buf() { return reinterpret_cast<float *>(spare() + kList); }
    static __device__ __forceinline__ uint4 *ring() { return reinterpret_cast<uint4 *>(spare() + kList); }
    // A bit a logit, and a word to spare at both ends (HELD: in the histogram's place).
    __device__ __forceinline__ uint32_t *penalised() const {
        return (HELD ? lo() : reinterpret_cast<uint32_t *>(buf() + a.slots)) + 1;
    }
    __device__ __forceinline__ uint32_t *ignored() const { return penalised() + a.words; }

    int tid, rank, ctas, searches = 0;
    int64_t row;
    const T *x;                       // this CTA's logits
    int start, count, phase, groups;  // its first, how many, offset of the first from a 16-byte boundary, 16-byte groups
    bool edits;                       // the row has penalised or ignored ids
    float top, lowest;                // largest and smallest logit above -inf
    float thread_top;                 // largest of this thread's
    float half_top, reach, slices;   // slices of a unit of (top - v) / 2, which has weight up to `reach`
    int bins;
    double wide_top, scale;
    enum { kPlain, kInfinite, kTiny } special;  // whether, and how, logits are not taken as they are
    bool limited = false;  // by top-k: tokens up to (limit_value, limit_index) in the order
    float limit_value;
    int limit_index;

    __device__ __forceinline__ bool leader() const { return rank == 0; }
    __device__ __forceinline__ void sync_all() {
        if (CLUSTER)
            cg::this_cluster().sync();
        else
            __syncthreads();
    }
    template <typename U>
    __device__ __forceinline__ U *at(U *mine, int cta) const {
        return CLUSTER ? cg::this_cluster().map_shared_rank(mine, cta) : mine;
    }

    // An empty histogram of that many slices.
    __device__ __forceinline__ void new_bins(int n) {
        bins = n;
        slices = fminf(__fdiv_rn(static_cast<float>(n - 1), reach), FLT_MAX);
        clear();
    }
    __device__ __forceinline__ void clear() {
        for (int i = 4 * tid; i < bins; i += 4 * kThreads) {
            *reinterpret_cast<uint4 *>(lo() + i) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4 *>(hi() + i) = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
    }

    // ---- the row -------------------------------------------------------------------------------------------
    static constexpr int L = 16 / sizeof(T);  // logits of a 16-byte group
    __device__ __forceinline__ bool ignores() const { return a.ignore && (a.streams > 0 ? row % a.streams == 0 : row == 0); }

    // The L bits of a group.
    __device__ __forceinline__ uint32_t bits_of(const uint32_t *words, int g) const {
        const int e = g * L - phase;
        return __funnelshift_r(words[e >> 5], words[(e >> 5) + 1], e & 31) & ((1u << L) - 1);
    }
    static __device__ __noinline__ float penalty_of(float v, float penalty) { return __fdiv_rn(v, penalty); }

    // A bit for every penalised and every ignored id of this CTA's share.
    __device__ __forceinline__ void mark_edits() {
        for (int i = tid - 1; i < 2 * a.words - 1; i += kThreads) penalised()[i] = 0;
        __syncthreads();
        if (a.recent)
            for (int64_t j = tid; j < a.recent_len; j += kThreads) {
                const int64_t id = a.recent[row * a.recent_len + j], e = id - start;
                if (id >= 0 && id < a.limit && e >= 0 && e < count) atomicOr(&penalised()[e >> 5], 1u << (e & 31));
            }
        if (ignores())
            for (int64_t j = tid; j < a.n_ignore; j += kThreads) {
                const int64_t e = a.ignore[j] - start;
                if (e >= 0 && e < count) atomicOr(&ignored()[e >> 5], 1u << (e & 31));
            }
        __syncthreads();
    }

    // f(group, logits, whole) for each of this CTA's groups (of those at both ends, what is not the CTA's is -inf);
    // `between` runs while the first loads are on their way.  The same threads take the same groups always.
    template <typename B, typename F>
    __device__ __forceinline__ void read_groups(B between, F f) {
        const int begin = phase > 0 ? 1 : 0, end = (phase + count) / L;  // whole groups
        const T *const base = x - phase;
        auto take = [&](const uint4 &raw, int g) {
            const T *values = reinterpret_cast<const T *>(&raw);
            float v[L];
#pragma unroll
            for (int i = 0; i < L; ++i) v[i] = to_float(values[i]);
            f(g, v, true);
        };
        if constexpr (HELD) {
            for (int g0 = begin + tid; g0 - tid < end || g0 == begin + tid; g0 += kAhead * kThreads) {
                uint4 raw[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
                    if (g0 + j * kThreads < end)
                        raw[j] = *reinterpret_cast<const uint4 *>(base + (g0 + j * kThreads) * L);
                if (g0 == begin + tid) between();
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    if (g0 + j * kThreads >= end) break;
                    take(raw[j], g0 + j * kThreads);
                }
            }
        } else {
            // a ring of kRing groups a thread in shared memory, which that thread alone fills and reads
            uint4 *const own = ring() + tid;
            auto start_copy = [&](int g, int slot) {
                if (g < end) cp_async16(own + slot * kThreads, base + g * L);
                cp_async_commit();
            };
#pragma unroll
            for (int j = 0; j < kRing; ++j) start_copy(begin + tid + j * kThreads, j);
            between();
            int slot = 0;
            for (int g = begin + tid; g < end; g += kThreads) {
                cp_async_wait_group<kRing - 1>();
                const uint4 raw = own[slot * kThreads];
                start_copy(g + kRing * kThreads, slot);
                slot = (slot + 1) % kRing;
                take(raw, g);
            }
            cp_async_wait_all();
        }
        // the parts of a group at both ends
        const int g = tid == 0 ? 0 : groups - 1;
        if ((tid == 0 && begin > 0) || (tid == kThreads - 1 && end < groups && (groups > 1 || begin == 0))) {
            float v[L];
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const int e = g * L - phase + i;
                v[i] = e >= 0 && e < count ? to_float(x[e]) : -INFINITY;
            }
            f(g, v, false);
        }
    }

    // Penalty and ignore list of a group read again.
    __device__ __forceinline__ void edit(float (&v)[L], int g) const {
        const uint32_t p = bits_of(penalised(), g), n = bits_of(ignored(), g);
        if (p | n) {
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (p >> i & 1) v[i] = penalty_of(v[i], a.penalty);
                if (n >> i & 1) v[i] = -INFINITY;
            }
        }
    }

    __device__ __forceinline__ void load() {
        start = rank * a.chunk;
        count = static_cast<int>(min(static_cast<int64_t>(a.chunk), a.vocab - start));
        x = static_cast<const T *>(a.logits) + row * a.ld + start;
        phase = static_cast<int>(reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (L - 1);
        groups = (phase + count + L - 1) / L;
        edits = a.recent || ignores();
        // Extremes: two instructions a logit that give NaN and -inf away where there is one, and then a second, careful
        // look at the thread's logits.
        float most = -INFINITY, least = INFINITY, quick_most = -INFINITY, quick_least = INFINITY;
        bool nan = false;
        auto note = [&](float v) {  // neither extreme takes a NaN, and the least no -inf
            nan |= isnan(v);
            most = fmaxf(most, v);
            least = fminf(least, v == -INFINITY ? INFINITY : v);
        };
        auto marks_of = [&](int g) { return edits ? bits_of(penalised(), g) | bits_of(ignored(), g) : 0u; };
        read_groups([&] { if (edits) mark_edits(); }, [&](int g, float(&v)[L], bool full) {
            if (HELD) {  // what is penalised or ignored is held as it came, and edited below
#pragma unroll
                for (int i = 0; i < L; i += 4)
                    *reinterpret_cast<float4 *>(buf() + g * L + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            } else if (edits) {
                edit(v, g);
            }
            const uint32_t marks = HELD ? marks_of(g) : 0;
            if (full && marks == 0) {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    asm("max.NaN.f32 %0, %0, %1;" : "+f"(quick_most) : "f"(v[i]));
                    quick_least = fminf(quick_least, v[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < L; ++i)
                    if (!(marks >> i & 1)) note(v[i]);
            }
        });
        if (isnan(quick_most) || quick_least == -INFINITY) {
            for (int g = (phase > 0 ? 1 : 0) + tid; g < (phase + count) / L; g += kThreads) {
                const uint32_t marks = HELD ? marks_of(g) : 0;
                for (int i = 0; i < L; ++i)
                    if (!(marks >> i & 1)) note(HELD ? buf()[g * L + i] : raw_logit(g * L + i - phase));
            }
        } else {
            most = fmaxf(most, quick_most), least = fminf(least, quick_least);
        }
        if (HELD && edits) {
            __syncthreads();
            float *const mine = buf() + phase;
            if (a.recent)
                for (int64_t j = tid; j < a.recent_len; j += kThreads) {
                    const int64_t id = a.recent[row * a.recent_len + j], e = id - start;
                    if (id < 0 || id >= a.limit || e < 0 || e >= count) continue;
                    const uint32_t bit = 1u << (e & 31);
                    if ((ignored()[e >> 5] & bit) || !(atomicAnd(&penalised()[e >> 5], ~bit) & bit)) continue;  // once an id
                    mine[e] = penalty_of(mine[e], a.penalty);
                    note(mine[e]);
                }
            if (ignores())
                for (int64_t j = tid; j < a.n_ignore; j += kThreads) {
                    const int64_t e = a.ignore[j] - start;
                    if (e >= 0 && e < count) mine[e] = -INFINITY;
                }
        }
        thread_top = most;
        const uint32_t most_key = __reduce_max_sync(0xffffffffu, key_of(most));
        const uint32_t least_key = __reduce_min_sync(0xffffffffu, key_of(least));
        nan = __any_sync(0xffffffffu, nan);
        // a place of its own for each warp: this barrier may be the kernel's first, so nothing could be set before it
        if ((tid & 31) == 0) {
            sh.warp_sums[tid >> 5] = (static_cast<u64>(most_key) << 32) | least_key;
            sh.warp_counts[tid >> 5] = nan;
        }
        __syncthreads();
    }

    // Largest and smallest key (and the NaN flag) of the row, from those of each warp and each CTA.
    __device__ __forceinline__ void share_extremes() {
        const int warp = tid & (kWarps - 1);
        uint32_t most = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(sh.warp_sums[warp] >> 32));
        uint32_t least = __reduce_min_sync(0xffffffffu, static_cast<uint32_t>(sh.warp_sums[warp]));
        int nan = __any_sync(0xffffffffu, sh.warp_counts[warp]);
        if (CLUSTER) {
            // Another CTA's shared memory may be touched once that CTA runs, which this barrier, the first, is what says:
            // so each leaves its own for the others to fetch.
            if (tid == 0) sh.own = {most, least, nan};
            sync_all();
            const Extremes theirs = *at(&sh.own, min(tid & 31, ctas - 1));
            most = __reduce_max_sync(0xffffffffu, theirs.most);
            least = __reduce_min_sync(0xffffffffu, theirs.least);
            nan = __any_sync(0xffffffffu, theirs.nan);
        }
        if (tid == 0) sh.nan = nan;
        top = value_of(most);
        lowest = value_of(least);
    }

    // This row's settings, by one thread ahead of the row.
    __device__ __forceinline__ void ask() {
        if (tid != kThreads - 1) return;
        Settings set{a.top_k_rows ? a.top_k_rows[row] : a.top_k,
                     a.temperature_rows ? a.temperature_rows[row] : a.temperature,
                     a.top_p_rows ? a.top_p_rows[row] : a.top_p, a.min_p_rows ? a.min_p_rows[row] : a.min_p,
                     a.uniforms[row], 0};
        float &t = set.temperature, &p = set.top_p, &m = set.min_p, &u = set.uniform;
        if (!(t >= 0.0f) || isinf(t)) set.bad = 1, t = 0.0f;
        if (set.top_k < 0) set.bad = 1, set.top_k = 0;
        if (set.top_k == 0 || set.top_k > a.vocab) set.top_k = a.vocab;
        if (!(p >= 0.0f && p <= 1.0f)) set.bad = 1, p = p < 0.0f ? 0.0f : 1.0f;
        if (!(m >= 0.0f && m <= 1.0f)) set.bad = 1, m = m > 1.0f ? 1.0f : 0.0f;
        if (!(u >= 0.0f && u < 1.0f)) set.bad = 1, u = u >= 1.0f ? 1.0f : 0.0f;
        if (t == 0.0f) set.top_k = 1;
        sh.set = set;
    }

    __device__ __forceinline__ void settings() {
        const float temperature = sh.set.temperature;
        scale = temperature > 0.0f ? kSteps * 1.4426950408889634074 / static_cast<double>(temperature) : 0.0;
        special = top == INFINITY ? kInfinite : temperature > 0.0f && temperature < kTinyTemperature ? kTiny : kPlain;
        if (special == kInfinite) top = lowest = 0.0f;
        // Half differences, so that none overflows.  The slices reach to the lowest logit, or to 31.9 T below the top,
        // where weights are below 2^-45 and round to nothing.
        half_top = 0.5f * top;
        wide_top = top;
        reach = fminf(__fmaf_rn(-0.5f, lowest, half_top), 15.95f * temperature);
        if (special) thread_top = seen(thread_top);
    }

    // A logit of a special row.  Beside +inf nothing else has weight: 0 among -inf.  At a tiny temperature the slices
    // would take in logits thousands of temperatures below the top: those are -inf.
    __device__ __forceinline__ float seen(float v) const {
        if (special == kInfinite) return v == INFINITY ? 0.0f : -INFINITY;
        return static_cast<double>(v) - wide_top >= -32.0 * static_cast<double>(sh.set.temperature) ? v : -INFINITY;
    }

    // Slice of a logit: never smaller for a smaller logit; `bins` and above where there is no weight (-inf among it)
    // and for NaN.  The sum with 2^23 leaves the nearest integer in the low bits.
    __device__ __forceinline__ uint32_t bin_of(float v) const {
        const float d = __fmaf_rn(-0.5f, v, half_top);
        return __float_as_uint(__fmaf_rn(d, slices, 8388608.0f)) - 0x4b000000u;
    }
    // A value below every logit of the slices up to `bin`: the lower edge, moved until it lies outside them.
    __device__ __forceinline__ float below(uint32_t bin) const {
        const float width = __fdiv_rn(2.0f, slices);
        for (float past = 1.0f; past < 100.0f; past *= 4.0f) {
            const float v = __fmaf_rn(-(static_cast<float>(bin) + past), width, top);
            if (bin_of(v) > bin) return v;
        }
        const float next = value_of(key_of(top) - 1);
        return bin_of(next) > bin ? next : -INFINITY;
    }
    // A value that no logit of the slices from `bin` on lies above.
    __device__ __forceinline__ float above(uint32_t bin) const {
        const float width = __fdiv_rn(2.0f, slices);
        for (uint32_t past = 1; past < min(bin, 100u); past *= 4) {
            const float v = __fmaf_rn(-static_cast<float>(bin - past), width, top);
            if (bin_of(v) < bin) return v;
        }
        return INFINITY;
    }
    __device__ __forceinline__ bool within(float v, int index) const {
        return !limited || v > limit_value || (v == limit_value && index <= limit_index);
    }
    __device__ __forceinline__ u64 weight(float v) const { return weight_of(v, wide_top, scale, sh.powers); }

    // f(logits, index of the first) for this CTA's tokens by fours.
    template <typename F>
    __device__ __forceinline__ void for_fours(F f) {
        auto four = [&](float(&v)[4], int first) {
            if (special) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = seen(v[i]);
            }
            f(v, first);
        };
        if constexpr (HELD) {
            const int quads = groups * L / 4;
            for (int g = tid; g < quads; g += kThreads) {
                const float4 q = reinterpret_cast<const float4 *>(buf())[g];
                float v[4] = {q.x, q.y, q.z, q.w};
                four(v, start + 4 * g - phase);
            }
        } else {
            read_groups([] {}, [&](int g, float(&group)[L], bool) {
                if (edits) edit(group, g);
#pragma unroll
                for (int i = 0; i < L; i += 4) {
                    float v[4] = {group[i], group[i + 1], group[i + 2], group[i + 3]};
                    four(v, start + g * L - phase + i);
                }
            });
        }
    }
    // f(logits, slices) for this CTA's tokens by fours; a token without weight, or beyond the limit of top-k, has a
    // slice of `bins` or above.
    template <typename F>
    __device__ __forceinline__ void for_slices(F f) {
        for_fours([&](const float(&v)[4], int first) {
            uint32_t bin[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) bin[i] = bin_of(v[i]);
            if (limited) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!within(v[i], first + i)) bin[i] = bins;
            }
            f(v, bin);
        });
    }

    // ---- histograms ----------------------------------------------------------------------------------------
    __device__ __forceinline__ void add(uint32_t bin, u64 w) {
        const uint32_t low = static_cast<uint32_t>(w);
        const uint32_t old = atomicAdd(&lo()[bin], low);
        const uint32_t high = static_cast<uint32_t>(w >> 32) + (old + low < old);
        if (high) atomicAdd(&hi()[bin], high);
    }

    __device__ __forceinline__ void add4(const uint32_t (&bin)[4], const u64 (&w)[4]) {
        uint32_t old[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (bin[i] < bins) old[i] = atomicAdd(&lo()[bin[i]], static_cast<uint32_t>(w[i]));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t high = static_cast<uint32_t>(w[i] >> 32) + (old[i] + static_cast<uint32_t>(w[i]) < old[i]);
            if (bin[i] < bins && high) atomicAdd(&hi()[bin[i]], high);
        }
    }

    // Running sums of the cluster's histogram, in the first CTA: a slice's words = what lies before it.
    __device__ __forceinline__ void running_sums() {
        sync_all();
        if (CLUSTER) {
            constexpr int kMost = kBins / 2 / kThreads;
            const int share = bins / ctas;
            u64 sum[kMost];
#pragma unroll
            for (int i = 0; i < kMost; ++i) {
                const int bin = rank * share + i * kThreads + tid;
                sum[i] = 0;
                if (i * kThreads + tid < share) {
#pragma unroll
                    for (int c = 0; c < kMaxCluster; ++c) {
                        const int from = min(c, ctas - 1);  // every load unconditional: all are on their way at once
                        const u64 part = (static_cast<u64>(*at(&hi()[bin], from)) << 32) + *at(&lo()[bin], from);
                        sum[i] += c < ctas ? part : 0;
                    }
                }
            }
            sync_all();
#pragma unroll
            for (int i = 0; i < kMost; ++i) {
                const int bin = rank * share + i * kThreads + tid;
                if (i * kThreads + tid < share) {
                    *at(&lo()[bin], 0) = static_cast<uint32_t>(sum[i]);
                    *at(&hi()[bin], 0) = static_cast<uint32_t>(sum[i] >> 32);
                }
            }
            sync_all();
        }
        if (!leader()) return;
        if (bins == kBins)
            add_up<kBins / kThreads>();
        else
            add_up<kCountBins / kThreads>();
    }

    // A thread's N neighbouring sums.
    template <int N>
    __device__ __forceinline__ void sums_of(u64 (&sum)[N]) const {
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const uint4 l = *reinterpret_cast<const uint4 *>(lo() + tid * N + i);
                const uint4 h = *reinterpret_cast<const uint4 *>(hi() + tid * N + i);
                sum[i] = (static_cast<u64>(h.x) << 32) | l.x, sum[i + 1] = (static_cast<u64>(h.y) << 32) | l.y;
                sum[i + 2] = (static_cast<u64>(h.z) << 32) | l.z, sum[i + 3] = (static_cast<u64>(h.w) << 32) | l.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] = (static_cast<u64>(hi()[tid * N + i]) << 32) | lo()[tid * N + i];
        }
    }
    template <int N>
    __device__ __forceinline__ void add_up() {
        u64 own[N], sum = 0, all;
        sums_of(own);
#pragma unroll
        for (int i = 0; i < N; ++i) sum += own[i];
        u64 before = sum_before(sum, all);
        uint32_t l[N], h[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            l[i] = static_cast<uint32_t>(before);
            h[i] = static_cast<uint32_t>(before >> 32);
            before += own[i];
        }
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                *reinterpret_cast<uint4 *>(lo() + tid * N + i) = make_uint4(l[i], l[i + 1], l[i + 2], l[i + 3]);
                *reinterpret_cast<uint4 *>(hi() + tid * N + i) = make_uint4(h[i], h[i + 1], h[i + 2], h[i + 3]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) lo()[tid * N + i] = l[i], hi()[tid * N + i] = h[i];
        }
        if (tid == 0) sh.total = all;
        __syncthreads();
    }

    // First CTA: the slice that `target` (below the total) falls into.
    template <int N>
    __device__ __forceinline__ void find_in(u64 target, Slice &to) {
        u64 sum[N];
        sums_of(sum);
        const u64 next = tid + 1 < kThreads ? (static_cast<u64>(hi()[(tid + 1) * N]) << 32) | lo()[(tid + 1) * N] : sh.total;
        if (sum[0] <= target && target < next) {
            to = {tid * N, sum[0], next};
#pragma unroll
            for (int i = 1; i < N; ++i) {
                if (sum[i] <= target)
                    to.bin = tid * N + i, to.before = sum[i];
                else
                    to.upto = min(to.upto, sum[i]);
            }
        }
        __syncthreads();
    }
    __device__ __forceinline__ void find(u64 target, Slice &to) {
        if (bins == kBins)
            find_in<kBins / kThreads>(target, to);
        else
            find_in<kCountBins / kThreads>(target, to);
    }
    // The first CTA's finds, told to the others.
    __device__ __forceinline__ void tell(u64 target) {
        if (leader() && tid < ctas) {
            Shared &to = *at(&sh, tid);
            to.target = target;
            if (tid > 0) to.slice = sh.slice, to.other = sh.other, to.joint = sh.joint;
        }
        sync_all();
    }
    __device__ __forceinline__ void locate(u64 target) {
        if (leader()) find(target, sh.slice);
        tell(target);
    }
    // After top-p's slice is found: the draw's slice, where it is the same whatever token of top-p's slice is the last.
    __device__ __forceinline__ void foresee() {
        if (!leader()) return;
        const u64 least = drawn(passed(sh.slice.before + 1)), most = drawn(passed(sh.slice.upto));
        find(least, sh.other);
        if (tid == 0) sh.joint = most < sh.other.upto;
        __syncthreads();
    }

    // Where the logits of slices [from, to] lie, and a little more: |v - middle| <= reach.  One subtraction a logit and
    // a minimum over four leave few quads to look at.
    struct Zone {
        float middle, reach;
    };
    __device__ __forceinline__ Zone zone(uint32_t from, uint32_t to) const {
        const float floor = below(to), ceiling = fminf(above(from), top);
        const float middle = 0.5f * floor + 0.5f * ceiling;
        if (isinf(floor)) return {0.0f, INFINITY};
        return {middle, fmaf(fabsf(middle), 1e-6f, 0.51f * ceiling - 0.51f * floor) + FLT_MIN};
    }
    static __device__ __forceinline__ bool near(const float (&v)[4], const Zone &z) {
        const float d = fminf(fminf(fabsf(v[0] - z.middle), fabsf(v[1] - z.middle)),
                              fminf(fabsf(v[2] - z.middle), fabsf(v[3] - z.middle)));
        return d <= z.reach;
    }

    // Collects the tokens whose slice lies in [from, to] and whose key in [low, high] in the first CTA's list; returns
    // how many there are (kList are held).
    __device__ __forceinline__ int collect(uint32_t from, uint32_t to, uint32_t low = 0, uint32_t high = 0xffffffffu) {
        uint32_t quads = 0;
        if constexpr (HELD) {
            const Zone z = zone(from, to);
            uint32_t bit = 1;
            for_fours([&](const float(&v)[4], int) {
                quads |= near(v, z) ? bit : 0;
                bit <<= 1;
            });
        }
        put(list(), from, to, low, high, quads);
        sync_all();
        return *at(&sh.cursor[searches++], 0);
    }
    // Both located slices, the second in the histogram's place.
    __device__ __forceinline__ void collect_both(int &n, int &other_n) {
        const uint32_t p = sh.slice.bin, d = sh.other.bin;
        uint32_t quads = 0, other_quads = 0;
        if constexpr (HELD) {
            const Zone z = zone(p, p), other = zone(d, d);
            uint32_t bit = 1;
            for_fours([&](const float(&v)[4], int) {
                quads |= near(v, z) ? bit : 0;
                other_quads |= near(v, other) ? bit : 0;
                bit <<= 1;
            });
        }
        if constexpr (HELD) {
#pragma unroll 1
            for (int i = 0; i < 2; ++i, ++searches)
                put(i ? reinterpret_cast<u64 *>(lo()) : list(), i ? d : p, i ? d : p, 0, 0xffffffffu,
                    i ? other_quads : quads);
        } else {
            const Zone z = zone(p, p), other = zone(d, d);
            for_fours([&](const float(&v)[4], int first) {
                if (!near(v, z) && !near(v, other)) return;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t bin = bin_of(v[i]);
                    if ((bin != p && bin != d) || !within(v[i], first + i)) continue;
                    for (int which = 0; which < 2; ++which) {
                        if (bin != (which ? d : p)) continue;
                        const int place = atomicAdd(at(&sh.cursor[searches + which], 0), 1);
                        if (place < kList)
                            at(which ? reinterpret_cast<u64 *>(lo()) : list(), 0)[place] = order_of(v[i], first + i);
                    }
                }
            });
            searches += 2;
        }
        sync_all();
        n = *at(&sh.cursor[searches - 2], 0);
        other_n = *at(&sh.cursor[searches - 1], 0);
    }

    // This CTA's tokens of slices [from, to] and keys [low, high] to the first CTA's list.  HELD: `quads` has a bit for
    // each of the thread's fours that can hold one; the threads' places come by a running sum.
    __device__ __forceinline__ void put(u64 *into, uint32_t from, uint32_t to, uint32_t low, uint32_t high, uint32_t quads) {
        int *const cursor = at(&sh.cursor[searches], 0);
        into = at(into, 0);
        auto member = [&](float v, int index) {
            const uint32_t key = key_of(v);
            return bin_of(v) - from <= to - from && key >= low && key <= high && within(v, index);
        };
        if constexpr (HELD) {
            static_assert(kMostHeld <= 64 * kThreads, "a bit for each of a thread's logits");
            u64 mine = 0;
            auto held = [&](int e) {
                const float v = buf()[e];
                return special ? seen(v) : v;
            };
            for (; quads != 0; quads &= quads - 1) {
                const int quad = __ffs(quads) - 1, e = 4 * (tid + quad * kThreads);
                for (int i = 0; i < 4; ++i)
                    if (member(held(e + i), start + e + i - phase)) mine |= 1ull << (4 * quad + i);
            }
            u64 all;
            int place = static_cast<int>(sum_before(static_cast<u64>(__popcll(mine)), all));
            if (CLUSTER) {
                if (tid == 0) sh.place = atomicAdd(cursor, static_cast<int>(all));
                __syncthreads();
                place += sh.place;
            } else if (tid == 0) {
                *cursor = static_cast<int>(all);
            }
            for (; mine != 0 && place < kList; mine &= mine - 1, ++place) {
                const int bit = __ffsll(mine) - 1, e = 4 * (tid + (bit >> 2) * kThreads) + (bit & 3);
                into[place] = order_of(held(e), start + e - phase);
            }
        } else {
            const Zone z = zone(from, to);
            for_fours([&](const float(&v)[4], int first) {
                if (!near(v, z)) return;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!member(v[i], first + i)) continue;
                    const int place = atomicAdd(cursor, 1);
                    if (place < kList) into[place] = order_of(v[i], first + i);
                }
            });
        }
    }

    // First CTA: the n listed tokens in order, one a thread (all ones behind them).  Up to a warp's: a bitonic network.
    // More: slices of the list's own range, each token's place is the slice's start and its rank in the slice (few
    // tokens, unless they are equal).  The histogram is not touched.
    __device__ __forceinline__ u64 sorted(u64 *list, int n) {
        u64 mine = tid < n ? list[tid] : ~0ull;
        if (n <= 32) {
            if (tid < 32) {
#pragma unroll
                for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
                    for (int stride = size >> 1; stride > 0; stride >>= 1) {
                        const u64 other = __shfl_xor_sync(0xffffffffu, mine, stride);
                        const bool smaller = ((tid & stride) == 0) == ((tid & size) == 0);
                        if ((other < mine) == smaller) mine = other;
                    }
            }
            return mine;
        }
        const uint32_t key = static_cast<uint32_t>(mine >> 32);  // ascending in the order
        const uint32_t first = __reduce_min_sync(0xffffffffu, key);
        const uint32_t last = __reduce_max_sync(0xffffffffu, tid < n ? key : 0u);
        if (tid == 0) sh.block_least = 0xffffffffu, sh.block_most = 0u;
        sh.places[tid] = 0;
        __syncthreads();
        if ((tid & 31) == 0) atomicMin(&sh.block_least, first), atomicMax(&sh.block_most, last);
        __syncthreads();
        const float half_first = 0.5f * value_of(~sh.block_least);
        const float per_unit = fminf(__fdiv_rn(static_cast<float>(kThreads - 1),
                                               __fmaf_rn(-0.5f, value_of(~sh.block_most), half_first)), FLT_MAX);
        const float d = __fmaf_rn(-0.5f, value_of(~key), half_first);
        const int part = tid < n ? min(kThreads - 1, static_cast<int>(d * per_unit)) : 0;
        if (tid < n) atomicAdd(&sh.places[part], 1);
        __syncthreads();
        const int own = sh.places[tid];
        u64 all;
        const int before = static_cast<int>(sum_before(static_cast<u64>(own), all));
        sh.places[tid] = before;
        sh.ends[tid] = before;
        __syncthreads();
        if (tid < n) spare()[atomicAdd(&sh.ends[part], 1)] = mine;
        __syncthreads();
        int place = 0;
        if (tid < n) {
            const int from = sh.places[part], to = sh.ends[part];
            place = from;
            for (int i = from; i < to; ++i) place += spare()[i] < mine;
            list[place] = mine;
        }
        __syncthreads();
        return tid < n ? list[tid] : ~0ull;
    }

    // Running sum over the CTA's threads (what lies before this one); `all`: the whole.
    __device__ __forceinline__ u64 sum_before(u64 own, u64 &all) {
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

    static __device__ __forceinline__ float value_in(u64 order) { return value_of(~static_cast<uint32_t>(order >> 32)); }
    static __device__ __forceinline__ int index_in(u64 order) { return static_cast<int>(static_cast<uint32_t>(order)); }

    // First CTA: which of the n listed tokens the target falls into.
    __device__ __forceinline__ void rank_list(u64 *list, int n, u64 before, u64 target, bool by_weight) {
        if (n <= 32) {  // a warp a token, or two: what lies before it is added up over the lanes
            const int lane = tid & 31;
            const u64 theirs = lane < n ? list[lane] : ~0ull;
            const u64 own = lane >= n ? 0 : by_weight ? weight(value_in(theirs)) : 1;
            for (int i = tid >> 5; i < n; i += kWarps) {
                const u64 mine = __shfl_sync(0xffffffffu, theirs, i);
                u64 sum = theirs < mine ? own : 0;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (lane == i && before + sum <= target && target < before + sum + own) sh.found = {mine, before + sum, own};
            }
        } else {
            const u64 mine = sorted(list, n);
            const u64 own = tid >= n ? 0 : by_weight ? weight(value_in(mine)) : 1;
            u64 all;
            const u64 sum = before + sum_before(own, all);
            if (sum <= target && target < sum + own) sh.found = {mine, sum, own};
        }
        __syncthreads();
    }

    // The token of the located slice that the target falls into: in the first CTA's sh.found.  A slice with too many
    // tokens costs the histogram (returns false then).
    __device__ __forceinline__ bool search_slice(bool by_weight) {
        const uint32_t slice = sh.slice.bin;
        u64 before = sh.slice.before;
        const u64 target = sh.target;
        uint32_t low_key = 0, high_key = 0xffffffffu;
        for (bool whole = true;; whole = false) {
            const int n = collect(slice, slice, low_key, high_key);
            if (n <= kList) {
                if (leader()) rank_list(list(), n, before, target, by_weight);
                return whole;
            }
            auto member = [&](float v, uint32_t bin) {
                const uint32_t key = key_of(v);
                return bin == slice && key >= low_key && key <= high_key;
            };
            // keys of the slice that is left
            uint32_t most = 0, least = 0xffffffffu, group = 0;
            if (tid == 0) sh.block_most = 0, sh.block_least = 0xffffffffu;
            __syncthreads();
            for_slices([&](const float(&v)[4], const uint32_t(&bin)[4]) {
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
            while (((most - least) >> shift) >= static_cast<uint32_t>(bins)) ++shift;
            clear();
            for_slices([&](const float(&v)[4], const uint32_t(&bin)[4]) {
                for (int i = 0; i < 4; ++i)
                    if (member(v[i], bin[i])) add((most - key_of(v[i])) >> shift, by_weight ? weight(v[i]) : 1);
            });
            running_sums();
            locate(target - before);
            before += sh.slice.before;
            high_key = most - (static_cast<uint32_t>(sh.slice.bin) << shift);
            low_key = max(least, high_key - ((1u << shift) - 1));
        }
    }

    // One of this CTA's logits, penalised and ignored as it may be; and as the order sees it.
    __device__ __forceinline__ float raw_logit(int i) const {
        float v = HELD ? buf()[phase + i] : to_float(x[i]);
        if (!HELD && edits) {
            const uint32_t bit = 1u << (i & 31);
            if (penalised()[i >> 5] & bit) v = penalty_of(v, a.penalty);
            if (ignored()[i >> 5] & bit) v = -INFINITY;
        }
        return v;
    }
    __device__ __forceinline__ float logit(int i) const {
        const float v = raw_logit(i);
        return special ? seen(v) : v;
    }

    // Index of this CTA's n-th (from 0) token with that logit: in the thread that holds it, -1 in the others.
    __device__ __forceinline__ int nth(float value, uint32_t n) {
        uint32_t before = 0;
        int found = -1;
        for (int i0 = 0; i0 < count && before <= n; i0 += kThreads) {
            const int i = i0 + tid;
            const bool is = i < count && logit(i) == value;
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
    __device__ __forceinline__ u64 least_weight() const {
        return static_cast<u64>(ceil(static_cast<double>(sh.set.min_p) * 17592186044416.0));  // 2^44
    }

    __device__ __forceinline__ void count_slices() {
        for_slices([&](const float(&)[4], const uint32_t(&bin)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (bin[i] < bins) atomicAdd(&lo()[bin[i]], 1u);
        });
    }

    // The histogram of weights and its running sums; what min-p leaves of them to the first CTA.
    __device__ __forceinline__ void weigh() {
        const u64 least = least_weight();
        const bool counted = sh.set.min_p > 0.0f;
        u64 passing = 0;
        for_slices([&](const float(&v)[4], const uint32_t(&bin)[4]) {
            if (min(min(bin[0], bin[1]), min(bin[2], bin[3])) >= bins) return;
            u64 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = weight(bin[i] < bins ? v[i] : top);
            }
            if (counted) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (bin[i] < bins && w[i] >= least) passing += w[i];
            }
            add4(bin, w);
        });
        if (counted) {
            u64 all;
            sum_before(passing, all);
            if (tid == 0) at(&sh, 0)->passing[rank] = all;
        }
        running_sums();
    }

    // The weight whose token is drawn, and the one whose token is the last that top-p keeps.
    __device__ __forceinline__ u64 drawn(u64 kept) const {
        const u64 place = static_cast<u64>(static_cast<double>(sh.set.uniform) * static_cast<double>(kept));
        return min(place, kept - 1);
    }
    __device__ __forceinline__ u64 nucleus(u64 all) const {
        const u64 part = static_cast<u64>(ceil(static_cast<double>(sh.set.top_p) * static_cast<double>(all)));
        return max(part, u64(1)) - 1;
    }
    // First CTA: what min-p leaves of a kept weight (both filters keep a prefix).
    __device__ __forceinline__ u64 passed(u64 kept) const {
        if (!(sh.set.min_p > 0.0f)) return kept;
        u64 passing = 0;
        for (int c = 0; c < ctas; ++c) passing += sh.passing[c];
        return min(kept, passing);
    }

    // First CTA: all that can be drawn is in the list (n tokens and no more): filters and draw over it in order.
    __device__ __forceinline__ void sample_list(int n) {
        const u64 mine = sorted(list(), n);
        const u64 own = tid < min(static_cast<int64_t>(n), sh.set.top_k) ? weight(value_in(mine)) : 0;
        u64 kept, passing;
        const u64 before = sum_before(own, kept);
        if (sh.set.top_p < 1.0f) {
            const u64 target = nucleus(kept);
            if (before <= target && target < before + own) sh.total = before + own;
            __syncthreads();
            kept = sh.total;
        }
        if (sh.set.min_p > 0.0f) {
            sum_before(own >= least_weight() ? own : 0, passing);
            kept = min(kept, passing);
        }
        const u64 target = drawn(kept);
        if (before <= target && target < before + own) finish(mine, own, kept);
    }

    __device__ __forceinline__ void sample() {
        const int64_t top_k = sh.set.top_k;
        const bool has_top_p = sh.set.top_p < 1.0f;
        enum { kTopK, kTopP, kDraw } stage = top_k < a.vocab ? kTopK : has_top_p ? kTopP : kDraw;

        // Few candidates: the first CTA has them all.  A short vocabulary; the tokens down to the k-th largest of the
        // threads' largest; the tokens up to the k-th one's slice (or to the last slice with a token).
#pragma unroll 1
        for (int attempt = a.vocab <= kList ? 0 : stage != kTopK ? 3 : top_k <= kList ? 1 : 2; attempt < 3; ++attempt) {
            if (attempt != 1) sync_all();  // the histogram before has been read
            new_bins(kCountBins);
            int upto = bins - 1;
            if (attempt > 0) {
                if (attempt == 1) {
                    const uint32_t bin = bin_of(thread_top);
                    if (bin < bins) atomicAdd(&lo()[bin], 1u);
                } else {
                    count_slices();
                }
                running_sums();
                locate(leader() ? min(static_cast<u64>(top_k), sh.total) - 1 : 0);
                upto = sh.slice.bin;
                // the threads have fewer than k tokens of weight; the slices have too many
                if (attempt == 1 ? sh.target + 1 < static_cast<u64>(top_k) : sh.slice.upto > kList) continue;
            }
            const int n = collect(0, upto);
            if (n <= kList) {
                if (leader()) sample_list(n);
                return;
            }
        }

        // One search after the other, each for a target in the running sums of its histogram.
        bool located = stage == kTopK, fresh = false, both = true;
        u64 kept = 0;  // first CTA: weight that top-p keeps
        if (located && sh.target + 1 < static_cast<u64>(top_k)) located = false, stage = has_top_p ? kTopP : kDraw;
        if (!located) fresh = true;
        for (;;) {
            if (fresh) {
                sync_all();  // the histogram before has been read
                new_bins(kBins);
                weigh();
                if (leader() && stage == kTopP) kept = sh.total;
                if (leader() && stage == kDraw && !has_top_p) kept = sh.total;
            }
            if (!located) {
                u64 target = 0;
                if (leader()) target = stage == kTopP ? nucleus(kept) : drawn(passed(kept));
                const bool try_both = stage == kTopP && both;
                if (leader()) find(target, sh.slice);
                if (try_both) foresee();
                tell(target);
                if (try_both && sh.joint) {
                    int n, other_n;
                    collect_both(n, other_n);
                    if (n <= kList && other_n <= kList) {
                        if (leader()) draw_both(n, other_n);
                        return;
                    }
                    both = false, fresh = true;  // one at a time then: a list has taken the histogram's place
                    continue;
                }
            }
            located = false;
            const bool whole = search_slice(stage != kTopK);
            if (stage == kDraw) break;
            if (stage == kTopK) {
                if (CLUSTER) {
                    if (leader() && tid > 0 && tid < ctas) at(&sh, tid)->found = sh.found;
                    sync_all();
                }
                limited = true;
                limit_value = value_in(sh.found.order);
                limit_index = index_in(sh.found.order);
                stage = has_top_p ? kTopP : kDraw;
                fresh = true;
            } else {
                if (leader()) kept = sh.found.before + sh.found.own;
                stage = kDraw;
                fresh = !whole;
            }
        }
        if (leader() && tid == 0) finish(sh.found.order, sh.found.own, passed(kept));
    }

    // First CTA: top-p's token, then the draw's, of the two lists.
    __device__ __forceinline__ void draw_both(int n, int other_n) {
        u64 kept = 0;
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            rank_list(i ? reinterpret_cast<u64 *>(lo()) : list(), i ? other_n : n, i ? sh.other.before : sh.slice.before,
                      i ? drawn(kept) : sh.target, true);
            if (i == 0) kept = passed(sh.found.before + sh.found.own);
            __syncthreads();
        }
        if (tid == 0) finish(sh.found.order, sh.found.own, kept);
    }

    // One thread of the first CTA: the token and its share of what was kept.
    __device__ __forceinline__ void finish(u64 order, u64 own, u64 kept) {
        a.out[row] = index_in(order);
        if (a.logprob)
            a.logprob[row] = static_cast<float>(log(static_cast<double>(own) / static_cast<double>(kept)));
        flag(0);
    }
    __device__ __forceinline__ void flag(int flags) {
        if (sh.set.bad) flags |= LEVO_SAMPLE_PARAM;
        if (sh.nan) flags |= LEVO_SAMPLE_NAN;
        if (a.status && flags) atomicOr(a.status, flags);
    }
};

template <typename T, bool CLUSTER, bool HELD>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
    __shared__ Shared shared;
    Row<T, CLUSTER, HELD> row(a, shared);
    row.run(CLUSTER ? blockIdx.x / cg::this_cluster().num_blocks() : blockIdx.x);
}

template <typename T>
int launch_sample(SampleArgs &a, const char *what, cudaStream_t stream) {
    constexpr int L = 16 / sizeof(T);
    // A CTA's tables, its share of the row in shared memory, and whether that leaves room for a second CTA on the SM.
    constexpr size_t rest = 2 * kBins * sizeof(uint32_t) + 2 * kList * sizeof(u64);
    static_assert(rest + kRing * kThreads * 16 + 2 * (kMaxVocab / 32 + 2) * sizeof(uint32_t) + sizeof(Shared) <= kHalfAnSm,
                  "two CTAs an SM read their rows again, whatever is edited");
    auto chunk_of = [&](int ctas) { return static_cast<int>((a.vocab + ctas - 1) / ctas + 7) / 8 * 8; };
    auto slots_of = [&](int ctas) { return (chunk_of(ctas) + 2 * L + 3) / 4 * 4; };
    auto two_an_sm = [&](int ctas) { return rest + slots_of(ctas) * sizeof(float) + sizeof(Shared) <= kHalfAnSm; };
    // One CTA a row up to kOneShare logits (three rows of 16385: one CTA each 10.2 us, two 13.2, four 12.6, since a
    // cluster's barriers cost more than its shorter passes save).  A longer row is split until its shares fit two an SM
    // (5 rows of 50257: four CTAs each 27.8 us, two 32.7; one row of 131072: eight 26.8, four 37.6), as far as the SMs
    // take all CTAs at once.
    int ctas = 1;
    while (ctas < kMaxCluster && a.rows * ctas * 2 <= 2LL * sm_count() &&
           (ctas == 1 ? a.vocab >= kOneShare : !two_an_sm(ctas)))
        ctas *= 2;
    a.chunk = chunk_of(ctas);
    a.words = a.recent || a.ignore ? (a.chunk + 31) / 32 + 2 : 0;
    // A share that leaves room for a second CTA is held in shared memory (192 rows of 16385: 14.6 us; read again, 18.9),
    // a longer one where every CTA has an SM of its own (100 rows of 20011: 18.3 us, read again 24.2; one row of 32000:
    // 20.9 and 24.9).  Others are read again from L2 (128 rows of 131072: two CTAs a row that read again 102 us, eight
    // that hold their shares 153, four rounds of clusters).
    a.slots = slots_of(ctas);
    const bool held = two_an_sm(ctas) || (a.rows * ctas <= sm_count() && a.slots <= kMostHeld);
    if (!held) a.slots = kRing * kThreads * 4;
    if (a.rows * ctas > 0x7fffffff)
        return set_error(LEVO_OPS_EUNSUPPORTED, std::string(what) + ": too many rows for one call");
    // Above 48 KB with the static part the kernel has to opt in, which resident_ctas does from the dynamic part alone.
    size_t smem = rest + a.slots * sizeof(float) + (held ? 0 : 2 * a.words * sizeof(uint32_t));
    if (smem + sizeof(Shared) > 48 * 1024) smem = std::max<size_t>(smem, 48 * 1024 + 16);
    auto *const kernel = ctas > 1 ? (held ? sample_kernel<T, true, true> : sample_kernel<T, true, false>)
                                  : (held ? sample_kernel<T, false, true> : sample_kernel<T, false, false>);
    int per_sm = 0;
    if (resident_ctas(reinterpret_cast<const void *>(kernel), kThreads, smem, &per_sm) != cudaSuccess)
        return check_launch(what);
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
    (void)cudaLaunchKernelEx(&cfg, kernel, a);
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
                       s.status, 0, 0, 0};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (s.dtype == LEVO_DTYPE_F32) return launch_sample<float>(a, w, st);
    if (s.dtype == LEVO_DTYPE_F16) return launch_sample<__half>(a, w, st);
    return launch_sample<__nv_bfloat16>(a, w, st);
}

}  // extern "C"
