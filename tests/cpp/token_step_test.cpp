// The token-step operators through include/levo_ops.hpp: known answers and the LM's exceptions.
// Built and run by tests/test_gpu_cpp_token_step.py on a GPU box.
#include <cmath>
#include <cstdio>
#include <stdexcept>
#include <string>
#include <vector>

#include <cuda_runtime.h>

#include "levo_ops.hpp"

static int failures = 0;
#define CHECK(cond)                                                                \
    do {                                                                           \
        if (!(cond)) {                                                             \
            std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            ++failures;                                                            \
        }                                                                          \
    } while (0)

template <class T>
static T *to_device(const std::vector<T> &h) {
    T *d = nullptr;
    cudaMalloc(&d, h.size() * sizeof(T) + 16);
    cudaMemcpy(d, h.data(), h.size() * sizeof(T), cudaMemcpyHostToDevice);
    return d;
}
template <class T>
static std::vector<T> to_host(const T *d, size_t n) {
    std::vector<T> h(n);
    cudaDeviceSynchronize();
    cudaMemcpy(h.data(), d, n * sizeof(T), cudaMemcpyDeviceToHost);
    return h;
}
template <class F>
static std::string message_of(F f) {
    try {
        f();
    } catch (const std::runtime_error &e) {
        return e.what();
    }
    return "";
}

int main() {
    using namespace levo::b200;

    // One head of four values at position 5, theta {1, 0.01}: pairs (0, 2) and (1, 3), or (0, 1) and (2, 3).
    const std::vector<double> theta = rope_theta(4);
    CHECK(theta.size() == 2 && theta[0] == 1.0 && std::fabs(theta[1] - 0.01) < 1e-17);
    const std::vector<float> x = {1.0F, 2.0F, 3.0F, 4.0F};
    double *dtheta = to_device(theta);
    float *dx = to_device(x), *dy = to_device(std::vector<float>(4)), *dback = to_device(std::vector<float>(4));
    for (const bool interleaved : {false, true}) {
        levo_rope r{};
        r.q = {dx, dy, 1, {4, 4, 4}, {4, 4, 4}};
        r.batch = r.tokens = 1;
        r.head_dim = r.rotary_dim = 4;
        r.theta = dtheta;
        r.start = 5;
        r.dtype = LEVO_DTYPE_F32;
        r.flags = interleaved ? LEVO_ROPE_INTERLEAVED : 0u;
        r.magnitude = 1.0F;
        rope_qk(r);
        const std::vector<float> y = to_host(dy, 4);
        for (int i = 0; i < 2; ++i) {
            const int a = interleaved ? 2 * i : i, b = interleaved ? 2 * i + 1 : i + 2;
            const double phi = 5.0 * theta[i];
            CHECK(std::fabs(y[a] - (x[a] * std::cos(phi) - x[b] * std::sin(phi))) < 2e-6);
            CHECK(std::fabs(y[b] - (x[a] * std::sin(phi) + x[b] * std::cos(phi))) < 2e-6);
        }
        r.q.in = dy;
        r.q.out = dback;
        r.flags |= LEVO_ROPE_ADJOINT;  // of a rotation: back
        rope_qk(r);
        const std::vector<float> back = to_host(dback, 4);
        for (int i = 0; i < 4; ++i) CHECK(std::fabs(back[i] - x[i]) < 4e-6);
        r.rotary_dim = 3;
        CHECK(message_of([&] { rope_qk(r); }).rfind("LeVo LM: levo_rope_qk: rotary_dim", 0) == 0);
    }

    // A cache of three rows that holds one: the token goes to row 1, rows 0 and 2 stay.
    const std::vector<float> cache(12, 7.0F);
    float *dk = to_device(cache), *dv = to_device(cache);
    int64_t *dlen = to_device(std::vector<int64_t>{1});
    levo_rope_append p{};
    p.rope.q = {dx, dy, 1, {4, 4, 4}, {4, 4, 4}};
    p.rope.k = {dx, dk, 1, {4, 4, 4}, {12, 4, 4}};
    p.v = {dx, dv, 1, {4, 4, 4}, {12, 4, 4}};
    p.rope.batch = p.rope.tokens = 1;
    p.rope.head_dim = p.rope.rotary_dim = p.v_dim = 4;
    p.rope.theta = dtheta;
    p.rope.dtype = LEVO_DTYPE_F32;
    p.rope.magnitude = 1.0F;
    p.capacity = 3;
    p.lengths = dlen;
    rope_append_kv(p);
    const std::vector<float> k = to_host(dk, 12), v = to_host(dv, 12);
    for (int i = 0; i < 4; ++i) {
        CHECK(k[i] == 7.0F && k[8 + i] == 7.0F && v[i] == 7.0F && v[8 + i] == 7.0F && v[4 + i] == x[i]);
        const int j = i % 2, a = j, b = j + 2;
        const double c = std::cos(theta[j]), s = std::sin(theta[j]);
        CHECK(std::fabs(k[4 + i] - (i < 2 ? x[a] * c - x[b] * s : x[a] * s + x[b] * c)) < 2e-6);
    }
    p.lengths = nullptr;
    CHECK(message_of([&] { rope_append_kv(p); }).find("lengths is null") != std::string::npos);

    // log 1, log 2, log 5 (of 8): in order 5/8, 2/8, 1/8.
    const std::vector<float> logits = {std::log(1.0F), std::log(2.0F), std::log(5.0F)};
    std::vector<float> rows;
    for (int i = 0; i < 4; ++i) rows.insert(rows.end(), logits.begin(), logits.end());
    float *dl = to_device(rows), *du = to_device(std::vector<float>{0.0F, 0.6F, 0.7F, 0.9F});
    int64_t *dt = to_device(std::vector<int64_t>(4, -1));
    float *dp = to_device(std::vector<float>(4));
    levo_sampling s{};
    s.logits = dl;
    s.rows = 4;
    s.vocab = s.ld = 3;
    s.uniforms = du;
    s.tokens_out = dt;
    s.logprob_out = dp;
    s.temperature = s.top_p = s.penalty = 1.0F;
    s.dtype = LEVO_DTYPE_F32;
    sample_tokens(s);
    CHECK((to_host(dt, 4) == std::vector<int64_t>{2, 2, 1, 0}));
    CHECK(std::fabs(to_host(dp, 4)[3] - std::log(0.125)) < 1e-6);
    s.top_k = 2;  // 5/7, 2/7
    sample_tokens(s);
    CHECK((to_host(dt, 4) == std::vector<int64_t>{2, 2, 2, 1}));
    s.top_p = 2.0F;
    CHECK(message_of([&] { sample_tokens(s); }).rfind("LeVo LM: levo_sample_tokens: top_p", 0) == 0);

    if (failures == 0) std::printf("token step ok\n");
    return failures ? 1 : 0;
}
