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

namespace levo {
namespace {

constexpr int kThreads = 256;

// sin and cos of f quarter turns, |f| <= 1/2: f * S(f^2) and C(f^2), the Taylor
// coefficients (pi/2)^k / k! of the two functions.  The first term left out is
// (pi/4)^11 / 11! = 1.8e-9 of the sine and (pi/4)^12 / 12! = 1.1e-10 of the cosine.
constexpr double kHalfPi = 1.57079632679489661923;
constexpr double quarter_coefficient(int k) {
    double c = 1.0;
    for (int i = 1; i <= k; ++i) c *= kHalfPi / i;
    return c;
}

struct Turn {
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
};

// One thread per (token, head, unit): a unit is a pair, or one copied value.
template <typename T>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeArgs<T> a) {
    const int64_t half = a.rotary_dim / 2;
    const int64_t units_qk = half + (a.head_dim - a.rotary_dim);
    const int64_t units = units_qk > a.v_dim ? units_qk : a.v_dim;
    const int64_t heads = a.q.heads + a.k.heads + a.v.heads;
    const int64_t total = a.batch * a.tokens * heads * units;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t u = i % units;
        int64_t head = i / units % heads;
        const int64_t token = i / (units * heads);
        const int64_t b = token / a.tokens, s = token % a.tokens;
        const bool is_q = head < a.q.heads;
        const bool is_v = head >= a.q.heads + a.k.heads;
        const Side<T> &side = is_q ? a.q : is_v ? a.v : a.k;
        head -= is_q ? 0 : is_v ? a.q.heads + a.k.heads : a.q.heads;
        if (u >= (is_v ? a.v_dim : units_qk)) continue;
        int64_t row = s;
        int64_t position = a.start + s;
        if (a.append) {
            const int64_t at = a.lengths[b] + s;
            position += at - s;
            if (!is_q) {
                const int64_t given = a.counts ? a.counts[b] : a.tokens;
                if ((given < 0 || given > a.tokens) && a.status) atomicOr(a.status, LEVO_APPEND_BAD_COUNT);
                if (s >= given) continue;
                if (at < 0 || at >= a.capacity) {
                    if (a.status) atomicOr(a.status, LEVO_APPEND_NO_ROOM);
                    continue;
                }
                row = at;
            }
        }
        if (a.positions) position = a.positions[b * a.ps[0] + s * a.ps[1]];
        const T *in = side.in + b * side.is[0] + s * side.is[1] + head * side.is[2];
        T *out = side.out + b * side.os[0] + row * side.os[1] + head * side.os[2];
        if (is_v) {
            out[u] = in[u];
        } else if (u >= half) {
            const int64_t d = a.rotary_dim + (u - half);
            out[d] = in[d];
        } else {
            const int64_t d1 = a.interleaved ? 2 * u : u;
            const int64_t d2 = a.interleaved ? 2 * u + 1 : u + half;
            const Turn t = turn_at(static_cast<double>(position), a.theta[u], a.magnitude, a.adjoint != 0);
            const float x1 = to_f32(in[d1]), x2 = to_f32(in[d2]);
            out[d1] = from_f32<T>(x1 * t.c - x2 * t.s);
            out[d2] = from_f32<T>(x1 * t.s + x2 * t.c);
        }
    }
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
    a.v_dim = ap ? ap->v_dim : 0;
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
    const int64_t units = std::max(r.rotary_dim / 2 + (r.head_dim - r.rotary_dim), a.v_dim);
    const int64_t total = r.batch * r.tokens * (a.q.heads + a.k.heads + a.v.heads) * units;
    const int64_t grid = std::min<int64_t>((total + kThreads - 1) / kThreads, int64_t(1) << 30);
    rope_kernel<T><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a);
    return check_launch(what);
}

constexpr int64_t kMaxSize = int64_t(1) << 31;  // of a batch, a token count, a head count or a dimension
constexpr int64_t kMaxSpan = int64_t(1) << 60;  // of a stride times its size
constexpr double kMaxWork = 1e16;               // values of one call: its counters stay inside 64 bits

// Whether [n0][n1][n2][inner] by these strides names distinct elements, and by how much it spans
// (sorted by stride, each dimension steps past all that the smaller ones reach).
bool distinct_elements(const int64_t (&stride)[3], const int64_t (&size)[3], int64_t inner) {
    int64_t reach = inner;
    bool done[3] = {false, false, false};
    for (int round = 0; round < 3; ++round) {
        int least = -1;
        for (int i = 0; i < 3; ++i)
            if (!done[i] && (least < 0 || stride[i] < stride[least])) least = i;
        done[least] = true;
        if (size[least] <= 1) continue;
        if (stride[least] < reach) return false;
        reach += stride[least] * (size[least] - 1);
    }
    return true;
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
    if (!distinct_elements(t.out_stride, out_size, dim)) return fail(": the output's strides overlap");
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

int dispatch(const levo_rope &r, const levo_rope_append *ap, const char *what, levo_stream_t stream) {
    const double width = static_cast<double>(std::max(r.head_dim, ap ? ap->v_dim : 0));
    const double heads = static_cast<double>(r.q.heads + r.k.heads + (ap ? ap->v.heads : 0));
    if (static_cast<double>(r.batch) * static_cast<double>(r.tokens) * heads * width > kMaxWork)
        return set_error(LEVO_OPS_EUNSUPPORTED, std::string(what) + ": too many values for one call");
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
    return dispatch(r, nullptr, w, stream);
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
    if ((r.k.heads && r.k.in == r.k.out) || (p.v.heads && p.v.in == p.v.out))
        return fail(": a cache may not be its own input");
    if (p.lengths == nullptr) return fail(": lengths is null");
    if (!aligned_to(p.lengths, 8) || !aligned_to(p.counts, 8) || !aligned_to(p.status, 4))
        return fail(": pointer is not aligned to its element size");
    if (r.batch == 0 || r.tokens == 0 || r.q.heads + r.k.heads + p.v.heads == 0) return LEVO_OPS_OK;
    return dispatch(r, append, w, stream);
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
