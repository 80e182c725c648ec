// Drives include/ops/{linear_attention,sandwich_norm}.h and their gradients the way a caller's block does: known answers small enough to be
// written down, refusals as exceptions. Built with hipcc by __graft_entry__.build(); run by tests/test_linear_interface.py on the GPU.
#include <cmath>
#include <cstdio>
#include <functional>
#include <stdexcept>
#include <string>
#include <vector>

#include "ops/backward/linear_attention_backward.h"
#include "ops/backward/sandwich_norm_backward.h"

namespace {

int failures = 0;

void expect(bool ok, const std::string& what) {
    if (!ok) {
        ++failures;
        std::printf("FAIL %s\n", what.c_str());
    }
}
Tensor device(std::vector<std::size_t> shape, const std::vector<float>& values) {
    Tensor t(std::move(shape), DeviceType::GPU, Dtype::F32);
    t.copy_from_host(values);
    return t;
}
std::vector<float> host(const Tensor& t) {
    if (hipDeviceSynchronize() != hipSuccess) throw std::runtime_error("synchronize failed");
    std::vector<float> values(t.numel());
    t.copy_to_host(values);
    return values;
}
bool close(const std::vector<float>& got, const std::vector<float>& want, float tolerance) {
    if (got.size() != want.size()) return false;
    for (std::size_t i = 0; i < got.size(); ++i)
        if (!(std::fabs(got[i] - want[i]) <= tolerance)) return false;
    return true;
}
template <typename E>
bool throws(const std::function<void()>& call) {
    try {
        call();
    } catch (const E&) {
        return true;
    } catch (...) {
        return false;
    }
    return false;
}

void linear() {
    // Two tokens, one head of two, a decay of 1/2: S = k1 v1' / 2 + k2 v2' behind the second.
    FlashAttentionOptions options;
    options.num_query_heads = options.num_kv_heads = 1;
    options.head_dim = 2;
    options.attention_scale = 1.0f;
    Tensor q = device({1, 2, 1, 2}, {1, 0, 1, 2}), k = device({1, 2, 1, 2}, {2, 4, 1, 0}), v = device({1, 2, 1, 2}, {1, 3, 5, 7});
    Tensor decay = device({1}, {std::log(0.5f)}), out = Tensor::zeros({1, 2, 1, 2}), state = Tensor::zeros({1, 1, 2, 2});
    linear_attention_forward(out, &state, q, k, v, decay, nullptr, nullptr, options);
    expect(close(host(out), {2, 6, 10, 22}, 1e-5f), "linear_attention_forward");  // (1 + 4) (1, 3) + 1 (5, 7)
    expect(close(host(state), {6, 10, 2, 6}, 1e-5f), "linear_attention_forward state");
    // The third token from that state, in place: S = (6, 10; 2, 6) / 2 + (1, 1)' (2, 0).
    Tensor q3 = device({1, 1, 1, 2}, {1, -1}), k3 = device({1, 1, 1, 2}, {1, 1}), v3 = device({1, 1, 1, 2}, {2, 0}), o3 = Tensor::zeros({1, 1, 1, 2});
    Tensor next = Tensor::zeros({1, 1, 2, 2});
    linear_attention_step(o3, next, state, q3, k3, v3, decay, nullptr, options);
    expect(close(host(next), {5, 5, 3, 3}, 1e-5f) && close(host(o3), {2, 2}, 1e-5f), "linear_attention_step");
    linear_attention_step(o3, state, state, q3, k3, v3, decay, nullptr, options);
    expect(host(state) == host(next), "linear_attention_step in place");
    Tensor again = Tensor::zeros({1, 1, 2, 2}), start = device({1, 1, 2, 2}, {6, 10, 2, 6});
    linear_attention_forward(o3, &again, q3, k3, v3, decay, &start, nullptr, options);
    expect(close(host(again), {5, 5, 3, 3}, 1e-5f) && close(host(o3), {2, 2}, 1e-5f), "linear_attention_forward from a state");
    // dO = (0, 0), (1, 0): dq2 = S (1, 0)' of the second token, dv2 = (q2.k2) dO, dv1 = (q2.k1) / 2 dO, dk2 = (v2.dO) q2, dk1 half of (v1.dO) q2.
    Tensor dout = device({1, 2, 1, 2}, {0, 0, 1, 0}), dq = Tensor::zeros({1, 2, 1, 2}), dk = Tensor::zeros({1, 2, 1, 2}),
           dv = Tensor::zeros({1, 2, 1, 2}), dstate = Tensor::zeros({1, 1, 2, 2});
    linear_attention_backward(dq, dk, dv, &dstate, dout, nullptr, q, k, v, decay, nullptr, nullptr, options);
    expect(close(host(dq), {0, 0, 6, 2}, 1e-5f), "linear_attention_backward query");
    expect(close(host(dk), {0.5f, 1, 5, 10}, 1e-5f), "linear_attention_backward key");
    expect(close(host(dv), {5, 0, 1, 0}, 1e-5f), "linear_attention_backward value");
    expect(close(host(dstate), {0.25f, 0, 0.5f, 0}, 1e-5f), "linear_attention_backward state");
    linear_attention_backward(dq, dk, dv, nullptr, dout, nullptr, q, k, v, decay, nullptr, nullptr, options, true);
    expect(close(host(dv), {10, 0, 2, 0}, 1e-5f), "linear_attention_backward accumulated");
    FlashAttentionOptions open = options;
    open.causal = false;
    Tensor two = Tensor::zeros({2});
    expect(throws<std::invalid_argument>([&] { linear_attention_forward(out, nullptr, q, k, v, decay, nullptr, nullptr, open); }), "not causal");
    expect(throws<std::invalid_argument>([&] { linear_attention_forward(out, nullptr, q, k, v, two, nullptr, nullptr, options); }), "decay's shape");
    expect(throws<std::invalid_argument>([&] { linear_attention_forward(out, &two, q, k, v, decay, nullptr, nullptr, options); }), "state's shape");
    expect(throws<std::invalid_argument>([&] { linear_attention_forward(o3, &start, q3, k3, v3, decay, &start, nullptr, options); }),
           "the initial state's place");
    expect(throws<std::invalid_argument>([&] { linear_attention_step(out, next, state, q, k, v, decay, nullptr, options); }), "two tokens");
}

void sandwich() {
    // f = (3, -3) is (1, -1) normed; x' = x / 2 + gate (1, -1) u; epsilon is far below a rounding.
    const float eps = 1e-12f;
    Tensor x = device({2, 2}, {2, 4, 2, 4}), f = device({2, 2}, {3, -3, 3, -3}), u = device({2}, {1, 2}), w = device({2}, {10, 100});
    Tensor gate = device({2, 2}, {1, 1, 2, 0}), stream = Tensor::zeros({2, 2}), y = Tensor::zeros({2, 2});
    sandwich_norm_forward(stream, y, x, f, u, &gate, w, 0.5f, eps);
    expect(close(host(stream), {2, 0, 3, 2}, 1e-5f), "sandwich_norm_forward stream");
    const float r2 = std::sqrt(2.0f), r = std::sqrt(6.5f);
    expect(close(host(y), {10 * r2, 0, 30 / r, 200 / r}, 1e-4f), "sandwich_norm_forward normed");
    sandwich_norm_forward(stream, y, x, f, u, nullptr, w, 0.5f, eps);
    expect(close(host(stream), {2, 0, 2, 0}, 1e-5f), "sandwich_norm_forward without a gate");
    // With nothing from the norm (dy = 0) the stream's gradient goes to x scaled, to the gate and u as it is.
    sandwich_norm_forward(stream, y, x, f, u, &gate, w, 0.5f, eps);
    Tensor ds = device({2, 2}, {4, 6, 8, 2}), dy = Tensor::zeros({2, 2}), dx = Tensor::zeros({2, 2}), df = Tensor::zeros({2, 2}),
           du = Tensor::zeros({2}), dgate = Tensor::zeros({2, 2}), dw = Tensor::zeros({2});
    sandwich_norm_backward(dx, df, du, &dgate, dw, &ds, dy, stream, f, u, &gate, w, 0.5f, eps);
    expect(close(host(dx), {2, 3, 4, 1}, 1e-5f), "sandwich_norm_backward stream");
    expect(close(host(dgate), {4, -12, 8, -4}, 1e-4f), "sandwich_norm_backward gate");
    expect(close(host(du), {20, -6}, 1e-4f) && close(host(dw), {0, 0}, 1e-5f), "sandwich_norm_backward weights");
    // df = (h - n mean(h n)) / 3, n = (1, -1), h = gate u G = (4, 12), (16, 0).
    expect(close(host(df), {8.0f / 3, 8.0f / 3, 8.0f / 3, 8.0f / 3}, 1e-4f), "sandwich_norm_backward branch");
    Tensor wide = Tensor::zeros({3}), gates = Tensor::zeros({3, 2});
    expect(throws<std::invalid_argument>([&] { sandwich_norm_forward(stream, y, x, f, wide, &gate, w, 0.5f, eps); }), "weight's shape");
    expect(throws<std::invalid_argument>([&] { sandwich_norm_forward(stream, y, x, f, u, &gates, w, 0.5f, eps); }), "gate's rows");
    expect(throws<std::invalid_argument>([&] { sandwich_norm_forward(stream, y, x, f, u, &gate, w, 0.5f, 0.0f); }), "epsilon");
    expect(throws<std::invalid_argument>([&] { sandwich_norm_backward(dx, df, du, &dgate, dw, &ds, dy, stream, f, u, nullptr, w, 0.5f, eps); }),
           "a gradient without a gate");
}

}  // namespace

int main() {
    try {
        linear();
        sandwich();
    } catch (const std::exception& error) {
        std::printf("FAIL unexpected exception: %s\n", error.what());
        ++failures;
    }
    std::printf("%d failure(s)\n", failures);
    return failures == 0 ? 0 : 1;
}
