// Drives include/ops/{layernorm,dropout,differential_attention}.h and their gradients the way a caller's block does: known answers
// small enough to be written down, one mask in both directions, refusals as exceptions. Built with hipcc by
// __graft_entry__.build(); run by tests/test_branch_interface.py on the GPU.
#include <cmath>
#include <cstdio>
#include <functional>
#include <stdexcept>
#include <string>
#include <vector>

#include "ops/backward/differential_attention_backward.h"
#include "ops/backward/dropout_backward.h"
#include "ops/backward/layernorm_backward.h"
#include "ops/layernorm.h"

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

void layernorm() {
    // Rows (1, 3) and (-2, 2): means 2 and 0, deviations 1 and 2; epsilon is far below a rounding of them.
    const float eps = 1e-12f;
    Tensor x = device({2, 2}, {1, 3, -2, 2}), w = device({2}, {2, 3}), b = device({2}, {10, 20}), y = Tensor::zeros({2, 2});
    layernorm_forward(y, x, w, b, eps);
    expect(close(host(y), {8, 23, 8, 23}, 1e-5f), "layernorm_forward");
    layernorm_forward(y, x, w, eps);
    expect(close(host(y), {-2, 3, -2, 3}, 1e-6f), "layernorm_forward without a bias");
    // A gradient of a row of two: g - mean(g) is odd in the row, and so is xh: nothing is left but the residual.
    Tensor dy = device({2, 2}, {1, 2, 3, 5}), dx = device({2, 2}, {7, 8, 9, 10}), dw = Tensor::zeros({2}), db = Tensor::zeros({2});
    layernorm_backward(dx, dw, &db, dy, x, w, eps, nullptr, &dx);
    expect(close(host(dx), {7, 8, 9, 10}, 1e-5f), "layernorm_backward on a residual in place");
    expect(close(host(dw), {-4, 7}, 1e-5f) && close(host(db), {4, 7}, 0), "layernorm_backward weight and bias");
    layernorm_backward(dx, dw, nullptr, dy, x, w, eps);
    expect(close(host(dx), {0, 0, 0, 0}, 1e-5f), "layernorm_backward without a bias");
    Tensor wide = device({3}, {1, 1, 1});
    expect(throws<std::invalid_argument>([&] { layernorm_forward(y, x, wide, eps); }), "layernorm_forward weight shape");
    expect(throws<std::invalid_argument>([&] { layernorm_forward(y, x, w, 0.0f); }), "layernorm_forward epsilon");
    expect(throws<std::invalid_argument>([&] { layernorm_backward(dx, dw, &wide, dy, x, w, eps); }), "layernorm_backward bias shape");
}

void dropout() {
    const std::vector<float> values(1001, 3.0f);
    Tensor x = device({7, 143}, values), out = Tensor::zeros({7, 143}), dx = Tensor::zeros({7, 143});
    DropoutOptions options;
    options.probability = 0.25f;  // kept values are multiplied by 4/3
    options.seed = 12345;
    dropout_forward(out, x, nullptr, options);
    dropout_backward(dx, x, nullptr, options);
    const std::vector<float> forward = host(out);
    expect(forward == host(dx), "dropout: one mask in both directions");
    std::size_t kept = 0;
    bool only = true;
    for (const float v : forward) {
        kept += v != 0.0f;
        only = only && (v == 0.0f || v == 4.0f);
    }
    expect(only && kept > 650 && kept < 850, "dropout: zeros and scaled values");  // 751 on average, deviation 14
    dropout_forward(out, x, x, nullptr, options);
    std::vector<float> onto(forward);
    for (float& v : onto) v += 3.0f;
    expect(host(out) == onto, "dropout onto a residual");
    dropout_backward(dx, x, nullptr, options, true);
    std::vector<float> twice(forward);
    for (float& v : twice) v *= 2.0f;
    expect(host(dx) == twice, "dropout_backward accumulated");
    // A counter on the device stands for the same counter value in the options.
    Tensor counter({2}, DeviceType::GPU, Dtype::F32);
    const std::uint64_t moved = 5;
    counter.copy_raw_from_host({reinterpret_cast<const std::uint8_t*>(&moved), sizeof(moved)});
    DropoutOptions by_counter = options, by_offset = options;
    by_counter.counter = static_cast<const std::uint64_t*>(counter.raw_data());
    by_offset.offset = moved;
    dropout_forward(out, x, nullptr, by_counter);
    dropout_forward(dx, x, nullptr, by_offset);
    expect(host(out) == host(dx) && host(out) != forward, "dropout: a counter on the device");
    options.probability = 2.0f;
    expect(throws<std::invalid_argument>([&] { dropout_forward(out, x, nullptr, options); }), "dropout probability");
    Tensor shorter = Tensor::zeros({7, 142});
    expect(throws<std::invalid_argument>([&] { dropout_forward(shorter, x); }), "dropout shape");
}

void differential() {
    FlashAttentionOptions options;
    options.num_query_heads = options.num_kv_heads = 1;
    options.head_dim = 2;
    options.attention_scale = 1.0f;
    // One query of two keys that it scores alike in the second map; in the first the second key weighs e times as much.
    const float e = std::exp(1.0f), first = 1.0f / (1.0f + e);
    options.query_position_offset = 1;
    Tensor q = device({1, 1, 1, 2}, {1, 1}), k = device({1, 2, 1, 2}, {0, 1, 1, 1}), v = device({1, 2, 1, 2}, {1, 2, 3, 5});
    Tensor lambda = device({1}, {0.5f}), out = Tensor::zeros({1, 1, 1, 2}), second = Tensor::zeros({1, 1, 1, 2}), lse = Tensor::zeros({2, 1, 1, 1});
    differential_attention_forward(out, second, lse, q, k, v, lambda, nullptr, options);
    const float o1[2] = {first * 1 + (1 - first) * 3, first * 2 + (1 - first) * 5}, o2[2] = {2, 3.5f};
    expect(close(host(out), {o1[0] - 1.0f, o1[1] - 1.75f}, 1e-5f), "differential_attention_forward");
    expect(close(host(second), {o2[0], o2[1]}, 1e-6f), "differential_attention_forward second map");
    expect(close(host(lse), {std::log(1 + e), 1.0f + std::log(2.0f)}, 1e-6f), "differential_attention_forward logsumexp");
    Tensor alone = Tensor::zeros({1, 1, 1, 2});
    differential_attention_forward(alone, q, k, v, lambda, nullptr, options);
    expect(host(alone) == host(out), "differential_attention_forward alone");
    Tensor dout = device({1, 1, 1, 2}, {1, 0}), dq = Tensor::zeros({1, 1, 1, 2}), dk = Tensor::zeros({1, 2, 1, 2}),
           dv = Tensor::zeros({1, 2, 1, 2}), dlambda = Tensor::zeros({1});
    differential_attention_backward(dq, dk, dv, dlambda, dout, out, second, lse, q, k, v, lambda, nullptr, options);
    const float ds = first * (1 - first) * 2.0f;  // of the first map's second key; the first key's is its negative
    expect(close(host(dq), {ds, 0.0f}, 1e-5f), "differential_attention_backward query");
    expect(close(host(dk), {-ds, 0.25f, ds, -0.25f}, 1e-5f), "differential_attention_backward key");
    expect(close(host(dv), {first - 0.25f, 0, 1 - first - 0.25f, 0}, 1e-6f), "differential_attention_backward value");
    expect(close(host(dlambda), {-2.0f}, 1e-5f), "differential_attention_backward lambda");
    differential_attention_backward(dq, dk, dv, dlambda, dout, out, second, lse, q, k, v, lambda, nullptr, options, true);
    expect(close(host(dlambda), {-4.0f}, 1e-5f) && close(host(dq), {2 * ds, 0.0f}, 1e-5f), "differential_attention_backward accumulated");

    Tensor q1 = device({1, 2}, {1, 2}), k1 = device({1, 2}, {0.5f, 0.25f}), q2 = device({1, 2}, {1, -1}), k2 = device({1, 2}, {3, 3});
    Tensor lambdas = Tensor::zeros({2});
    differential_lambda_forward(lambdas, q1, k1, q2, k2, 0.75f);  // e^1 - e^0 + 0.75
    expect(close(host(lambdas), {e - 0.25f, e - 0.25f}, 1e-6f), "differential_lambda_forward");
    Tensor dlambdas = device({2}, {1, 2}), g1 = Tensor::zeros({1, 2}), g2 = Tensor::zeros({1, 2}), g3 = Tensor::zeros({1, 2}),
           g4 = Tensor::zeros({1, 2});
    differential_lambda_backward(g1, g2, g3, g4, dlambdas, q1, k1, q2, k2);
    expect(close(host(g1), {1.5f * e, 0.75f * e}, 1e-5f) && close(host(g2), {3 * e, 6 * e}, 1e-5f) && close(host(g3), {-9, -9}, 1e-5f) &&
               close(host(g4), {-3, 3}, 1e-5f),
           "differential_lambda_backward");
    FlashAttentionOptions odd = options;
    odd.head_dim = 3;
    Tensor q3 = Tensor::zeros({1, 1, 1, 3}), k3 = Tensor::zeros({1, 2, 1, 3});
    expect(throws<std::invalid_argument>([&] { differential_attention_forward(q3, q3, k3, k3, lambda, nullptr, odd); }), "an odd head");
    expect(throws<std::invalid_argument>([&] { differential_attention_forward(alone, q, k, v, lambdas, nullptr, options); }), "lambda's size");
    expect(throws<std::invalid_argument>([&] { differential_lambda_forward(lambda, lambdas, k1, q2, k2, 0.0f); }), "vectors' shapes");
}

}  // namespace

int main() {
    try {
        layernorm();
        dropout();
        differential();
    } catch (const std::exception& error) {
        std::printf("FAIL unexpected exception: %s\n", error.what());
        ++failures;
    }
    std::printf("%d failure(s)\n", failures);
    return failures == 0 ? 0 : 1;
}
