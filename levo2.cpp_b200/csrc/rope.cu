// Rotary positions on q and k, and the same with the append to the KV cache.
//
// A pair (x1, x2) of a head at position p turns by phi = p * theta:
//   y1 = m (x1 cos phi - x2 sin phi),  y2 = m (x1 sin phi + x2 cos phi);
// the adjoint turns by -phi.  Every value is read and written once, a pair
// costs six F32 operations and its share of one sine and cosine: the HBM bounds
// all but the smallest calls.
//
// The phase.  p * theta grows to 1e6 radians and more, of which only the
// fraction of a turn matters, so it is formed in F64 in quarter turns:
// h = p * (theta * 2/pi) as the unevaluated sum of a product and its FMA
// remainder, n the nearest integer (whose two lowest bits are the quadrant), and
// f = h - n in [-1/2, 1/2], rounded to F32 only then.  sin and cos of f quarter
// turns are polynomials in f^2 (below) and the quadrant swaps and negates them.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "strided.h"

namespace levo {
namespace {

// sin and cos of f quarter turns, |f| <= 1/2: f * S(f^2) and C(f^2), the Taylor
// coefficients (pi/2)^k / k! of the two functions.  The first term left out is
// (pi/4)^11 / 11! = 1.8e-9 of the sine and (pi/4)^12 / 12! = 1.1e-10 of the cosine.
constexpr double kHalfPi = 1.57079632679489661923;
constexpr double quarter_coefficient(int k) {
    double c = 1.0;
    for (int i = 1; i <= k; ++i) c *= kHalfPi / i;
    return c;
}

struct alignas(8) Turn {
    float c, s;
};

__device__ __forceinline__ Turn turn_at(double position, double theta, float magnitude, bool adjoint) {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: the sum's ulp is 1
    const double quarters = theta * (1.0 / kHalfPi);
    const double h = position * quarters;
    const double rest = __fma_rn(position, quarters, -h);
    const double r = h + kRound;
    const int quadrant = __double2loint(r) & 3;
    const float f = static_cast<float>((h - (r - kRound)) + rest);
    const float z = f * f;
    float s = __fmaf_rn(z, static_cast<float>(quarter_coefficient(9)), -static_cast<float>(quarter_coefficient(7)));
    s = __fmaf_rn(s, z, static_cast<float>(quarter_coefficient(5)));
    s = __fmaf_rn(s, z, -static_cast<float>(quarter_coefficient(3)));
    s = __fmaf_rn(s, z, static_cast<float>(quarter_coefficient(1))) * f;
    float c = __fmaf_rn(z, -static_cast<float>(quarter_coefficient(10)), static_cast<float>(quarter_coefficient(8)));
    c = __fmaf_rn(c, z, -static_cast<float>(quarter_coefficient(6)));
    c = __fmaf_rn(c, z, static_cast<float>(quarter_coefficient(4)));
    c = __fmaf_rn(c, z, -static_cast<float>(quarter_coefficient(2)));
    c = __fmaf_rn(c, z, 1.0f);
    Turn t;
    t.c = (quadrant & 1) ? s : c;
    t.s = (quadrant & 1) ? c : s;
    if (quadrant == 1 || quadrant == 2) t.c = -t.c;
    if (quadrant >= 2) t.s = -t.s;
    if (adjoint) t.s = -t.s;
    t.c *= magnitude;
    t.s *= magnitude;
    return t;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

template <typename T>
struct Side {
    const T *in;
    T *out;
    int64_t heads;
    int64_t is[3], os[3];
};

template <typename T>
struct RopeArgs {
    Side<T> q, k, v;  // v: copied (append only)
    int64_t batch, tokens, head_dim, rotary_dim, v_dim;
    const double *theta;
    const int64_t *positions;
    int64_t ps[2];
    int64_t start;
    float magnitude;
    int interleaved, adjoint;
    // append
    int append;
    int64_t capacity;
    const int64_t *lengths, *counts;
    int32_t *status;
    // launch shape
    int turned_chunks, qk_chunks, v_chunks, chunks;  // of q and k that turn, of q and k, of v, the larger
    uint32_t all_tokens;
    int lane_chunks, heads_per_block, token_lanes, tile;
};

// VEC neighbouring values: one load or store.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
    T v[VEC];
};

// A head is cut into chunks of two vectors of VEC values, so that a pair never spans threads:
//   half layout:  vectors c and c + rotary_dim/2/VEC (the two members of VEC pairs);
//   interleaved:  vectors c and c + n of the 2n (or 2n-1) turned ones, VEC/2 pairs each;
//   values that are copied (behind rotary_dim, and v): vectors c and c + n of theirs.
// In every case neighbouring threads touch neighbouring vectors.
struct Chunk {
    int first, second;  // offsets in a head; second < 0: none
};

template <int VEC, bool INTER>
__device__ __forceinline__ Chunk turned_chunk(int c, int rotary_dim) {
    if (!INTER) return {c * VEC, rotary_dim / 2 + c * VEC};
    if (VEC == 1) return {2 * c, 2 * c + 1};
    const int vectors = rotary_dim / VEC, n = (vectors + 1) / 2;
    return {c * VEC, c + n < vectors ? (c + n) * VEC : -1};
}

template <int VEC>
__device__ __forceinline__ Chunk copied_chunk(int c, int from, int to) {
    const int vectors = (to - from) / VEC, n = (vectors + 1) / 2;
    return {from + c * VEC, c + n < vectors ? from + (c + n) * VEC : -1};
}

// Where pair p's cosine lies (its sine two floats on) among the floats of a token's turns: chunk c's VEC pairs are
// read as Turns2 c, c + turned_chunks, ... (neighbouring threads on neighbouring ones).
template <int VEC, bool INTER>
__device__ __forceinline__ int turn_slot(int p, int turned_chunks) {
    int c = p / VEC, j = p % VEC;
    if (INTER && VEC > 1) {
        constexpr int H = VEC > 1 ? VEC / 2 : 1;
        const int vector = p / H;
        const bool late = vector >= turned_chunks;
        c = late ? vector - turned_chunks : vector;
        j = p % H + (late ? H : 0);
    }
    return 4 * (j / 2 * turned_chunks + c) + j % 2;
}

// Two neighbouring values to F32 and back as one word of the 16-bit types (taken apart and put together again by
// halves they cost a 16001-token BF16 backward pass 10 %).
__device__ __forceinline__ float2 to_f32x2(const float *p) { return *reinterpret_cast<const float2 *>(p); }
__device__ __forceinline__ float2 to_f32x2(const __half *p) {
    return __half22float2(*reinterpret_cast<const __half2 *>(p));
}
__device__ __forceinline__ float2 to_f32x2(const __nv_bfloat16 *p) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(p));
}
__device__ __forceinline__ void from_f32x2(float2 v, float *p) { *reinterpret_cast<float2 *>(p) = v; }
__device__ __forceinline__ void from_f32x2(float2 v, __half *p) {
    *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(v.x, v.y);
}
__device__ __forceinline__ void from_f32x2(float2 v, __nv_bfloat16 *p) {
    *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(v.x, v.y);
}

// The turns of two pairs: cosines, then sines.
struct alignas(16) Turns2 {
    float2 c, s;
};

// One pair.  Explicit roundings: every vector width and layout gives the same bits.
__device__ __forceinline__ float2 turn_pair(float x1, float x2, float c, float s) {
    return make_float2(__fmaf_rn(x1, c, -__fmul_rn(x2, s)), __fmaf_rn(x1, s, __fmul_rn(x2, c)));
}

// Turns the VEC pairs that a thread's two vectors hold, two pairs at a time.  turns: the chunk's first Turns2 of the
// token, the others turned_chunks apart.
template <typename T, int VEC, bool INTER>
__device__ __forceinline__ void turn_pairs(Vec<T, VEC> (&x)[2], const Turns2 *turns, int turned_chunks) {
    if constexpr (VEC == 1) {
        const Turns2 t = turns[0];
        const float x1 = to_f32(x[0].v[0]), x2 = to_f32(x[1].v[0]);
        const float2 y = turn_pair(x1, x2, t.c.x, t.s.x);
        x[0].v[0] = from_f32<T>(y.x);
        x[1].v[0] = from_f32<T>(y.y);
    } else if constexpr (INTER) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const Turns2 t = turns[i / 2 * turned_chunks];
#pragma unroll
            for (int j = i; j < i + 2; ++j) {
                T *const pair = &x[j / (VEC / 2)].v[2 * (j % (VEC / 2))];
                const float2 v = to_f32x2(pair);
                const float c = j > i ? t.c.y : t.c.x, s = j > i ? t.s.y : t.s.x;
                from_f32x2(turn_pair(v.x, v.y, c, s), pair);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const Turns2 t = turns[i / 2 * turned_chunks];
            const float2 x1 = to_f32x2(x[0].v + i), x2 = to_f32x2(x[1].v + i);
            const float2 p = __fmul2_rn(x2, t.s);
            from_f32x2(__ffma2_rn(x1, t.c, make_float2(-p.x, -p.y)), x[0].v + i);
            from_f32x2(__ffma2_rn(x1, t.s, __fmul2_rn(x2, t.c)), x[1].v + i);
        }
    }
}

// 384 threads, three CTAs an SM (56 registers): 512 and two, 256 and four were 0 to 10 % slower over the sizes below.
constexpr int kMaxThreads = 384;
constexpr int kCtasPerSm = 3;
// Bytes that a thread has on their way: 128 (four tokens of two 16-byte vectors).  Half and twice that cost 5 % on
// a 4 x 2048-token prompt: fewer bytes in flight, and fewer, longer CTAs at the end.
constexpr int kBytesInFlight = 128;
// Turns of a CTA's tile: 32 KB of shared memory.  (A single token that turns more than 4096 values by one value an
// access, where a pair takes 16 bytes, has up to 64 KB to itself.)
constexpr int kMaxTurns = 4096;
constexpr int kMaxTile = 32;     // tokens of a CTA

// A token of the tile: where its values lie (element offsets of the first head of q, k and v; out < 0: k and v have no
// row in the caches), and its position.
struct Place {
    int64_t in[3], out[3];
    double position;
};

// One value vector, global to shared memory (asynchronously where the hardware copies that many bytes).
template <int BYTES>
__device__ __forceinline__ void copy_in(void *to, const void *from) {
    if constexpr (BYTES == 16) {
        cp_async16(to, from);
    } else if constexpr (BYTES >= 4) {
        const unsigned dst = static_cast<unsigned>(__cvta_generic_to_shared(to));
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(from), "n"(BYTES) : "memory");
    } else {
        *static_cast<uint16_t *>(to) = *static_cast<const uint16_t *>(from);
    }
}

// A CTA turns a tile of tokens.  A thread keeps one chunk of one head and goes through the tile's tokens: it starts
// the copies of all its vectors to shared memory (it alone reads them: no registers wait for them and no barrier), the
// CTA evaluates every sine and cosine of the tile once while they are on their way, and the thread turns and stores.
//
// Bound by HBM on long inputs: 16001 tokens of 40 BF16 heads of 128 take 52.5 us, 6.2 TB/s (95 % of the measured copy
// rate); 4 x 2048 tokens of 24 F16 heads 18.7 us, 5.4 TB/s (the start and end of 2048 CTAs and 220 instructions a
// warp and 32 bytes a lane, two thirds of the issue slots); 2 x 1000 tokens of 40 F32 heads of 110, cut head by head
// into 8 bytes an access, 16.5 us, 4.3 TB/s.  Held in registers instead of staged (two heads or tokens a thread), 4 x 2048
// tokens took 26 to 36 us: the values on their way cost the occupancy that hides them.  One token: 3 us, the launch.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kMaxThreads, kCtasPerSm) rope_kernel(const RopeArgs<T> a) {
    using V = Vec<T, VEC>;
    constexpr int kPairs2 = (VEC + 1) / 2;
    extern __shared__ __align__(16) unsigned char smem[];
    Turns2 *const turns = reinterpret_cast<Turns2 *>(smem);  // [tile token][kPairs2][turned chunk]
    V *const staged = reinterpret_cast<V *>(smem + a.tile * kPairs2 * a.turned_chunks * sizeof(Turns2));
    __shared__ Place places[kMaxTile];
    const uint32_t first_token = blockIdx.x * static_cast<uint32_t>(a.tile);
    const int tile = static_cast<int>(min(static_cast<uint32_t>(a.tile), a.all_tokens - first_token));
    const int q_end = static_cast<int>(a.q.heads), k_end = q_end + static_cast<int>(a.k.heads);
    const int half = static_cast<int>(a.rotary_dim) / 2;
    // Everything that the sines wait for is loaded first.
    const double first_theta = a.theta[threadIdx.x % half];
    int64_t row = 0, position = 0, given = a.tokens;
    int64_t b = 0, s = 0;
    if (threadIdx.x < tile) {
        const uint32_t token = first_token + threadIdx.x;
        b = token / static_cast<uint32_t>(a.tokens);
        s = token % static_cast<uint32_t>(a.tokens);
        if (a.append) row = a.lengths[b];
        if (a.counts) given = a.counts[b];
        if (a.positions) position = a.positions[b * a.ps[0] + s * a.ps[1]];
        Place &p = places[threadIdx.x];
        p.in[0] = b * a.q.is[0] + s * a.q.is[1];
        p.in[1] = b * a.k.is[0] + s * a.k.is[1];
        p.in[2] = b * a.v.is[0] + s * a.v.is[1];
    }
    __syncthreads();

    const int lane = static_cast<int>(threadIdx.x) % a.lane_chunks, group = static_cast<int>(threadIdx.x) / a.lane_chunks;
    const int head = static_cast<int>(blockIdx.y) * a.heads_per_block + group % a.heads_per_block;
    const int which = head < q_end ? 0 : head < k_end ? 1 : 2;
    const Side<T> &side = which == 0 ? a.q : which == 1 ? a.k : a.v;
    const int n = head - (which == 0 ? 0 : which == 1 ? q_end : k_end);
    const T *const in = side.in + n * side.is[2];
    T *const out = side.out + n * side.os[2];
    const int token_lane = group / a.heads_per_block;
    const bool active = token_lane < a.token_lanes && n < side.heads;
    V *const own = staged + threadIdx.x;
    for (int c0 = 0; c0 < a.chunks; c0 += a.lane_chunks) {
        const int c = c0 + lane;
        const bool turns_here = which < 2 && c < a.turned_chunks;
        Chunk part = {-1, -1};
        if (turns_here)
            part = turned_chunk<VEC, INTER>(c, 2 * half);
        else if (which < 2 && c < a.qk_chunks)
            part = copied_chunk<VEC>(c - a.turned_chunks, 2 * half, static_cast<int>(a.head_dim));
        else if (which == 2 && c < a.v_chunks)
            part = copied_chunk<VEC>(c, 0, static_cast<int>(a.v_dim));
        const int t0 = active && part.first >= 0 ? token_lane : tile;
        V *to = own;
        for (int t = t0; t < tile; t += a.token_lanes) {
            const T *const from = in + places[t].in[which];
            copy_in<sizeof(V)>(to, from + part.first);
            if (part.second >= 0) copy_in<sizeof(V)>(to + blockDim.x, from + part.second);
            to += 2 * blockDim.x;
        }
        if (c0 == 0) {
            if (threadIdx.x < tile) {
                row += s;
                if (!a.positions) position = a.start + row;
                bool taken = true;
                if (a.append) {
                    const bool room = row >= 0 && row < a.capacity;
                    taken = s < given && room;
                    if (a.status && blockIdx.y == 0) {
                        if (given < 0 || given > a.tokens) atomicOr(a.status, LEVO_APPEND_BAD_COUNT);
                        if (s < given && !room && a.k.heads + a.v.heads > 0) atomicOr(a.status, LEVO_APPEND_NO_ROOM);
                    }
                }
                Place &p = places[threadIdx.x];
                p.out[0] = b * a.q.os[0] + s * a.q.os[1];
                p.out[1] = taken ? b * a.k.os[0] + row * a.k.os[1] : -1;
                p.out[2] = taken ? b * a.v.os[0] + row * a.v.os[1] : -1;
                p.position = static_cast<double>(position);
            }
            __syncthreads();
            for (int i = threadIdx.x; i < tile * half; i += blockDim.x) {
                const int t = i / half, p = i - t * half;
                const Turn turn = turn_at(places[t].position, i < blockDim.x ? first_theta : a.theta[p], a.magnitude, a.adjoint != 0);
                float *const at = reinterpret_cast<float *>(turns + t * kPairs2 * a.turned_chunks) +
                                  turn_slot<VEC, INTER>(p, a.turned_chunks);
                at[0] = turn.c;
                at[2] = turn.s;
            }
            __syncthreads();
        }
        cp_async_wait_all();
        to = own;
        for (int t = t0; t < tile; t += a.token_lanes, to += 2 * blockDim.x) {
            const int64_t at = places[t].out[which];
            if (at < 0) continue;
            V x[2] = {to[0], to[blockDim.x]};
            if (turns_here) turn_pairs<T, VEC, INTER>(x, turns + t * kPairs2 * a.turned_chunks + c, a.turned_chunks);
            *reinterpret_cast<V *>(out + at + part.first) = x[0];
            if (part.second >= 0) *reinterpret_cast<V *>(out + at + part.second) = x[1];
        }
    }
}

// Values that every pointer, stride and extent of the call allows in one access (16 bytes at most).
template <typename T>
int vector_width(const RopeArgs<T> &a) {
    int vec = 16 / static_cast<int>(sizeof(T));
    auto fits = [&](const Side<T> &s, int64_t rows, int64_t dim) {
        if (s.heads == 0) return true;
        const int64_t in_size[3] = {a.batch, a.tokens, s.heads}, out_size[3] = {a.batch, rows, s.heads};
        bool ok = aligned_to(s.in, vec * sizeof(T)) && aligned_to(s.out, vec * sizeof(T)) && dim % vec == 0;
        for (int i = 0; i < 3; ++i)
            ok = ok && (in_size[i] <= 1 || s.is[i] % vec == 0) && (out_size[i] <= 1 || s.os[i] % vec == 0);
        return ok;
    };
    const int64_t rows = a.append ? a.capacity : a.tokens;
    for (; vec > 1; vec /= 2)
        if ((a.interleaved ? a.rotary_dim : a.rotary_dim / 2) % vec == 0 && fits(a.q, a.tokens, a.head_dim) &&
            fits(a.k, rows, a.head_dim) && fits(a.v, rows, a.v_dim))
            break;
    return vec;
}

template <typename T, int VEC>
int launch_width(RopeArgs<T> &a, const char *what, cudaStream_t stream) {
    constexpr int kPairs2 = (VEC + 1) / 2, kItems = std::min<int>(8, kBytesInFlight / (2 * sizeof(Vec<T, VEC>)));
    auto half_up = [](int64_t n) { return static_cast<int>((n + 1) / 2); };
    a.turned_chunks = a.interleaved && VEC > 1 ? half_up(a.rotary_dim / VEC) : static_cast<int>(a.rotary_dim / 2 / VEC);
    a.qk_chunks = a.turned_chunks + half_up((a.head_dim - a.rotary_dim) / VEC);
    a.v_chunks = half_up(a.v_dim / VEC);
    a.chunks = std::max(a.qk_chunks, a.v_chunks);
    const int64_t tokens = a.batch * a.tokens, heads = a.q.heads + a.k.heads + a.v.heads;
    if (tokens > INT32_MAX)
        return set_error(LEVO_OPS_EUNSUPPORTED, std::string(what) + ": too many tokens for one call");
    a.all_tokens = static_cast<uint32_t>(tokens);
    // Threads of a CTA: chunks x heads x token lanes; each goes through up to kItems tokens.
    a.lane_chunks = std::min(a.chunks, kMaxThreads);
    const int64_t enough = 2LL * sm_count();  // CTAs, before heads share one
    const int64_t fit = std::max<int64_t>(1, std::min<int64_t>(kMaxThreads / a.lane_chunks, tokens * heads / enough));
    const int64_t groups = (heads + fit - 1) / fit;
    a.heads_per_block = static_cast<int>((heads + groups - 1) / groups);
    const int64_t lanes = std::max(1, 256 / (a.lane_chunks * a.heads_per_block));
    const int per_token = kPairs2 * a.turned_chunks * static_cast<int>(sizeof(Turns2));
    const int64_t most = std::min<int64_t>({tokens, kMaxTile, std::max<int64_t>(1, kMaxTurns * 8 / per_token)});
    a.token_lanes = static_cast<int>(std::min(lanes, most));
    const int64_t items = std::max<int64_t>(1, std::min<int64_t>(kItems, tokens * groups / (a.token_lanes * 4LL * sm_count())));
    a.tile = static_cast<int>(std::min(most, a.token_lanes * items));
    const int threads = std::max(32, (a.lane_chunks * a.heads_per_block * a.token_lanes + 31) / 32 * 32);
    const int64_t blocks = (tokens + a.tile - 1) / a.tile;
    if (groups > 65535)
        return set_error(LEVO_OPS_EUNSUPPORTED, std::string(what) + ": too many heads for one call");
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(groups));
    const int passes = (a.tile + a.token_lanes - 1) / a.token_lanes;
    // Above 48 KB with the static part the kernel has to opt in, which resident_ctas does from the dynamic part alone.
    size_t smem = static_cast<size_t>(a.tile) * per_token + static_cast<size_t>(passes) * 2 * threads * sizeof(Vec<T, VEC>);
    auto *const kernel = a.interleaved ? rope_kernel<T, VEC, true> : rope_kernel<T, VEC, false>;
    if (smem + kMaxTile * sizeof(Place) > 48 * 1024) smem = std::max<size_t>(smem, 48 * 1024 + 16);
    int per_sm = 0;
    if (smem > 48 * 1024 && resident_ctas(reinterpret_cast<const void *>(kernel), threads, smem, &per_sm) != cudaSuccess)
        return check_launch(what);
    kernel<<<grid, threads, smem, stream>>>(a);
    return check_launch(what);
}

template <typename T>
int launch_rope(const levo_rope &r, const levo_rope_append *ap, const char *what, cudaStream_t stream) {
    auto side = [](const levo_rope_tensor &t) {
        Side<T> s{static_cast<const T *>(t.in), static_cast<T *>(t.out), t.heads, {}, {}};
        for (int i = 0; i < 3; ++i) {
            s.is[i] = t.in_stride[i];
            s.os[i] = t.out_stride[i];
        }
        return s;
    };
    RopeArgs<T> a{};
    a.q = side(r.q);
    a.k = side(r.k);
    if (ap) a.v = side(ap->v);
    a.batch = r.batch;
    a.tokens = r.tokens;
    a.head_dim = r.head_dim;
    a.rotary_dim = r.rotary_dim;
    a.v_dim = ap && ap->v.heads ? ap->v_dim : 0;
    a.theta = r.theta;
    a.positions = r.positions;
    a.ps[0] = r.position_stride[0];
    a.ps[1] = r.position_stride[1];
    a.start = r.start;
    a.magnitude = r.magnitude;
    a.interleaved = (r.flags & LEVO_ROPE_INTERLEAVED) ? 1 : 0;
    a.adjoint = (r.flags & LEVO_ROPE_ADJOINT) ? 1 : 0;
    if (ap) {
        a.append = 1;
        a.capacity = ap->capacity;
        a.lengths = ap->lengths;
        a.counts = ap->counts;
        a.status = ap->status;
    }
    switch (vector_width(a)) {
        case 8: return launch_width<T, 16 / sizeof(T) < 8 ? 4 : 8>(a, what, stream);
        case 4: return launch_width<T, 4>(a, what, stream);
        case 2: return launch_width<T, 2>(a, what, stream);
        default: return launch_width<T, 1>(a, what, stream);
    }
}

constexpr int64_t kMaxSize = int64_t(1) << 31;  // of a batch, a token count, a head count or a dimension
constexpr int64_t kMaxDim = 2 * kMaxTurns;      // a token's sines and cosines fit a CTA's shared memory
constexpr int64_t kMaxSpan = int64_t(1) << 60;  // of a stride times its size
constexpr double kMaxWork = 1e16;               // values of one call: its counters stay inside 64 bits

Strided input_of(const levo_rope_tensor &t, int64_t batch, int64_t tokens, int64_t dim) {
    return {reinterpret_cast<uintptr_t>(t.in), {t.in_stride[0], t.in_stride[1], t.in_stride[2]},
            {batch, tokens, t.heads}, dim};
}
Strided output_of(const levo_rope_tensor &t, int64_t batch, int64_t rows, int64_t dim) {
    return {reinterpret_cast<uintptr_t>(t.out), {t.out_stride[0], t.out_stride[1], t.out_stride[2]},
            {batch, rows, t.heads}, dim};
}

int check_tensor(const char *what, const char *name, const levo_rope_tensor &t, int64_t batch, int64_t tokens,
                 int64_t rows, int64_t dim, size_t element) {
    auto fail = [&](const char *why) {
        return set_error(LEVO_OPS_EINVAL, std::string(what) + ": " + name + why);
    };
    if (t.heads < 0 || t.heads >= kMaxSize) return fail(": bad head count");
    if (t.heads == 0 || batch == 0 || tokens == 0) return LEVO_OPS_OK;  // nothing is read or written
    if (t.in == nullptr || t.out == nullptr) return fail(": required pointer is null");
    if (!aligned_to(t.in, element) || !aligned_to(t.out, element))
        return fail(": pointer is not aligned to its element size");
    const int64_t in_size[3] = {batch, tokens, t.heads}, out_size[3] = {batch, rows, t.heads};
    for (int i = 0; i < 3; ++i) {
        if (t.in_stride[i] < 0 || t.out_stride[i] < 0) return fail(": negative stride");
        if (t.in_stride[i] > kMaxSpan / std::max<int64_t>(in_size[i], 1) ||
            t.out_stride[i] > kMaxSpan / std::max<int64_t>(out_size[i], 1))
            return fail(": stride too large");
    }
    if (!output_of(t, batch, rows, dim).distinct()) return fail(": the output's strides overlap");
    if (t.in == t.out && rows == tokens) {
        for (int i = 0; i < 3; ++i)
            if (in_size[i] > 1 && t.in_stride[i] != t.out_stride[i])
                return fail(": in place with other strides");
    }
    return LEVO_OPS_OK;
}

int check_rope(const char *what, const levo_rope &r, size_t *element) {
    auto fail = [&](const char *why) { return set_error(LEVO_OPS_EINVAL, std::string(what) + why); };
    switch (r.dtype) {
        case LEVO_DTYPE_F32: *element = 4; break;
        case LEVO_DTYPE_F16:
        case LEVO_DTYPE_BF16: *element = 2; break;
        default: return fail(": dtype must be F32, F16 or BF16");
    }
    if (r.batch < 0 || r.tokens < 0) return fail(": negative size");
    if (r.batch >= kMaxSize || r.tokens >= kMaxSize || r.head_dim >= kMaxSize) return fail(": size too large");
    if (r.rotary_dim < 2 || r.rotary_dim % 2 != 0 || r.rotary_dim > r.head_dim)
        return fail(": rotary_dim must be even and in [2, head_dim]");
    if (!std::isfinite(r.magnitude)) return fail(": magnitude must be finite");
    if (r.theta == nullptr) return fail(": theta is null");
    if (!aligned_to(r.theta, 8) || !aligned_to(r.positions, 8))
        return fail(": pointer is not aligned to its element size");
    if (r.positions != nullptr && (r.position_stride[0] < 0 || r.position_stride[1] < 0))
        return fail(": negative position stride");
    return LEVO_OPS_OK;
}

// Whether one token's input lies exactly on a row of its own cache: whatever row the token goes to, each thread reads
// and writes its own values of a head.
bool on_a_row(const Strided &in, const Strided &cache, size_t element) {
    for (int i : {0, 2})
        if (in.size[i] > 1 && in.stride[i] != cache.stride[i]) return false;
    const uintptr_t apart = (in.at - cache.at) / element;
    const int64_t rows = cache.size[1];
    return in.size[1] == 1 && rows > 1 && in.at >= cache.at && apart % static_cast<uintptr_t>(cache.stride[1]) == 0 &&
           apart / static_cast<uintptr_t>(cache.stride[1]) < static_cast<uintptr_t>(rows);
}

// Outputs that share elements with another tensor's output or input, or with their own input but in place: threads
// would race on them.
int check_overlaps(const char *what, const levo_rope &r, const levo_rope_append *ap, size_t element) {
    auto fail = [&](const char *why) { return set_error(LEVO_OPS_EINVAL, std::string(what) + why); };
    const levo_rope_tensor *const tensors[3] = {&r.q, &r.k, ap ? &ap->v : nullptr};
    Strided in[3], out[3];
    int n = 0;
    for (int i = 0; i < 3; ++i) {
        const levo_rope_tensor *const t = tensors[i];
        if (!t || !t->heads) continue;
        const int64_t dim = i == 2 ? ap->v_dim : r.head_dim;
        in[n] = input_of(*t, r.batch, r.tokens, dim);
        out[n++] = output_of(*t, r.batch, ap && i > 0 ? ap->capacity : r.tokens, dim);
    }
    for (int i = 0; i < n; ++i)
        for (int j = 0; j < n; ++j)
            if (i != j && ((i < j && overlap(out[i], out[j], element)) || overlap(out[i], in[j], element)))
                return fail(": an output overlaps another tensor's output or input");
    for (int i = 0; i < n; ++i) {
        if (in[i].at == out[i].at && in[i].size[1] == out[i].size[1]) continue;  // in place: check_tensor saw the strides
        if (overlap(out[i], in[i], element) && !on_a_row(in[i], out[i], element))
            return fail(": an output overlaps its own input and is not in place");
    }
    return LEVO_OPS_OK;
}

int dispatch(const levo_rope &r, const levo_rope_append *ap, size_t element, const char *what, levo_stream_t stream) {
    if (r.head_dim > kMaxDim || (ap && ap->v.heads && ap->v_dim > kMaxDim))
        return set_error(LEVO_OPS_EUNSUPPORTED, std::string(what) + ": head dimension above 8192");
    const double width = static_cast<double>(std::max(r.head_dim, ap ? ap->v_dim : 0));
    const double heads = static_cast<double>(r.q.heads + r.k.heads + (ap ? ap->v.heads : 0));
    if (static_cast<double>(r.batch) * static_cast<double>(r.tokens) * heads * width > kMaxWork)
        return set_error(LEVO_OPS_EUNSUPPORTED, std::string(what) + ": too many values for one call");
    const int rc = check_overlaps(what, r, ap, element);
    if (rc != LEVO_OPS_OK) return rc;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (r.dtype == LEVO_DTYPE_F32) return launch_rope<float>(r, ap, what, s);
    if (r.dtype == LEVO_DTYPE_F16) return launch_rope<__half>(r, ap, what, s);
    return launch_rope<__nv_bfloat16>(r, ap, what, s);
}

}  // namespace
}  // namespace levo

extern "C" {

LEVO_OPS_API int levo_rope_qk(const levo_rope *rope, levo_stream_t stream) {
    using namespace levo;
    clear_error();
    const char *w = "levo_rope_qk";
    if (rope == nullptr) return set_error(LEVO_OPS_EINVAL, std::string(w) + ": arguments are null");
    const levo_rope &r = *rope;
    size_t element = 0;
    int rc = check_rope(w, r, &element);
    if (rc != LEVO_OPS_OK) return rc;
    if (r.flags & ~(LEVO_ROPE_INTERLEAVED | LEVO_ROPE_ADJOINT))
        return set_error(LEVO_OPS_EINVAL, std::string(w) + ": unknown flag");
    if ((rc = check_tensor(w, "q", r.q, r.batch, r.tokens, r.tokens, r.head_dim, element)) != LEVO_OPS_OK) return rc;
    if ((rc = check_tensor(w, "k", r.k, r.batch, r.tokens, r.tokens, r.head_dim, element)) != LEVO_OPS_OK) return rc;
    if (r.batch == 0 || r.tokens == 0 || r.q.heads + r.k.heads == 0) return LEVO_OPS_OK;
    return dispatch(r, nullptr, element, w, stream);
}

LEVO_OPS_API int levo_rope_append_kv(const levo_rope_append *append, levo_stream_t stream) {
    using namespace levo;
    clear_error();
    const char *w = "levo_rope_append_kv";
    if (append == nullptr) return set_error(LEVO_OPS_EINVAL, std::string(w) + ": arguments are null");
    const levo_rope_append &p = *append;
    const levo_rope &r = p.rope;
    size_t element = 0;
    int rc = check_rope(w, r, &element);
    if (rc != LEVO_OPS_OK) return rc;
    auto fail = [&](const char *why) { return set_error(LEVO_OPS_EINVAL, std::string(w) + why); };
    if (r.flags & ~LEVO_ROPE_INTERLEAVED) return fail(": unknown flag (the adjoint does not append)");
    if (p.capacity < 0 || p.capacity >= kMaxSize) return fail(": bad capacity");
    if (p.v.heads != 0 && (p.v_dim < 1 || p.v_dim >= kMaxSize)) return fail(": bad v_dim");
    if ((rc = check_tensor(w, "q", r.q, r.batch, r.tokens, r.tokens, r.head_dim, element)) != LEVO_OPS_OK) return rc;
    if ((rc = check_tensor(w, "k", r.k, r.batch, r.tokens, p.capacity, r.head_dim, element)) != LEVO_OPS_OK) return rc;
    if ((rc = check_tensor(w, "v", p.v, r.batch, r.tokens, p.capacity, p.v_dim, element)) != LEVO_OPS_OK) return rc;
    if (r.tokens > 1 && ((r.k.heads && r.k.in == r.k.out) || (p.v.heads && p.v.in == p.v.out)))
        return fail(": a cache may not be its own input");
    if (p.lengths == nullptr) return fail(": lengths is null");
    if (!aligned_to(p.lengths, 8) || !aligned_to(p.counts, 8) || !aligned_to(p.status, 4))
        return fail(": pointer is not aligned to its element size");
    if (r.batch == 0 || r.tokens == 0 || r.q.heads + r.k.heads + p.v.heads == 0) return LEVO_OPS_OK;
    return dispatch(r, append, element, w, stream);
}

LEVO_OPS_API int levo_rope_theta_host(double *theta_host, int64_t rotary_dim, double base, int32_t scaling,
                                      double factor, double context, double slow, double fast) {
    using namespace levo;
    clear_error();
    const char *w = "levo_rope_theta_host";
    auto fail = [&](const char *why) { return set_error(LEVO_OPS_EINVAL, std::string(w) + why); };
    if (theta_host == nullptr) return fail(": required pointer is null");
    if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim >= kMaxSize) return fail(": rotary_dim must be even and at least 2");
    if (!std::isfinite(base) || !(base > 0.0)) return fail(": base must be finite and positive");
    if (scaling < LEVO_ROPE_SCALE_NONE || scaling > LEVO_ROPE_SCALE_BY_PARTS) return fail(": unknown scaling");
    if (scaling != LEVO_ROPE_SCALE_NONE && !(std::isfinite(factor) && factor >= 1.0))
        return fail(": factor must be finite and at least 1");
    if (scaling == LEVO_ROPE_SCALE_NTK && rotary_dim == 2) return fail(": NTK scaling needs a rotary_dim of 4 or more");
    if (scaling == LEVO_ROPE_SCALE_BY_PARTS) {
        if (!std::isfinite(context) || !(context > 0.0)) return fail(": context must be finite and positive");
        if (!std::isfinite(fast) || !(slow >= 0.0) || !(fast > slow)) return fail(": 0 <= slow < fast is required");
    }
    const double n = static_cast<double>(rotary_dim);
    if (scaling == LEVO_ROPE_SCALE_NTK) base *= std::pow(factor, n / (n - 2.0));
    if (!std::isfinite(base)) return fail(": the scaled base is not finite");
    for (int64_t i = 0; i < rotary_dim / 2; ++i) {
        double theta = std::pow(base, -2.0 * static_cast<double>(i) / n);
        if (scaling == LEVO_ROPE_SCALE_LINEAR) theta /= factor;
        if (scaling == LEVO_ROPE_SCALE_BY_PARTS) {
            const double turns = context * theta / (4.0 * kHalfPi);
            const double g = std::min(std::max((turns - slow) / (fast - slow), 0.0), 1.0);
            theta = (1.0 - g) * theta / factor + g * theta;
        }
        theta_host[i] = theta;
    }
    return LEVO_OPS_OK;
}

}  // extern "C"
