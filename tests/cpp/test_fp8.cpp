// test_fp8.cpp -- FP8 expert layers through the C++20 host layer: DeviceExpertLayer::quantizeFp8 and
// HipMoEBlock on such a layer.
//
//   test_fp8 cpu   argument checks; needs no GPU
//   test_fp8 gpu   the quantised layer byte for byte, and a block against the CPU oracle
#include "hm_backend.hpp"
#include "hm_moe.h"
#include "hm_moe_block.hpp"
#include "hm_tensor.hpp"

#include "hm_oracle.h"

#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <memory>
#include <span>
#include <stdexcept>
#include <string>
#include <vector>

extern "C" {
void hm_synth_normal(uint64_t seed, uint64_t tag, int64_t n, float mean, float std, float* out);
}

using namespace hm;
using tensor::DType;
using tensor::Shape;

namespace {

int g_checks = 0, g_failures = 0;

void expect(bool cond, const std::string& what) {
    ++g_checks;
    if (!cond) {
        ++g_failures;
        std::fprintf(stderr, "FAIL: %s\n", what.c_str());
    }
}

void expectInvalid(const std::function<void()>& f, const std::string& what) {
    bool thrown = false;
    try {
        f();
    } catch (const std::invalid_argument&) {
        thrown = true;
    }
    expect(thrown, what);
}

double e4m3(unsigned byte) {
    const int e = (byte >> 3) & 15, m = byte & 7;
    const double v = e ? std::ldexp(1.0 + m / 8.0, e - 7) : std::ldexp(m / 8.0, -6);
    return byte & 0x80 ? -v : v;
}

// The e4m3 byte nearest to v, |v| <= 448, ties to the even one.
unsigned nearest(double v) {
    const double a = std::fabs(v);
    unsigned best = 0;
    for (unsigned b = 1; b < 0x7f; ++b) {
        const double d = std::fabs(e4m3(b) - a), was = std::fabs(e4m3(best) - a);
        if (d < was || (d == was && b % 2 == 0)) best = b;
    }
    return best | (std::signbit(v) ? 0x80u : 0u);
}

constexpr std::size_t E = 3, H = 200, I = 136;

// A payload of bfloat16 values, so that the bytes are decided exactly.
std::vector<float> payload() {
    std::vector<float> p(E * 3 * H * I);
    hm_synth_normal(5, 1, (int64_t)p.size(), 0.0F, 0.05F, p.data());
    for (auto& v : p) {
        std::uint32_t u;
        std::memcpy(&u, &v, 4);
        u &= 0xffff0000u;
        std::memcpy(&v, &u, 4);
    }
    return p;
}

void cpuTests() {
    const auto p = payload();
    const auto bytes = std::as_bytes(std::span(p));
    expectInvalid([&] { (void)DeviceExpertLayer::quantizeFp8(nullptr, bytes, E, H, I); }, "no backend");
    expect(tensor::sizeOf(DType::FP8) == 1, "an FP8 value is a byte");
    expect(hm_fp8_pitch(H) == 256 && hm_fp8_pitch(I) == 256, "rows are padded to 128 bytes");
    expect(hm_packed_layer_bytes(E, H, I, HM_DTYPE_FP8) == E * (2 * I * 256 + H * 256), "layer bytes");
    expect(nearest(448.0) == 0x7e && nearest(-1.0) == 0xb8 && nearest(17.0) == 0x58 && nearest(19.0) == 0x5a,
           "the test's own rounding");
}

void gpuTests(const std::shared_ptr<backend::HipBackend>& hip) {
    const auto p = payload();
    const auto bytes = std::as_bytes(std::span(p));
    expectInvalid([&] { (void)DeviceExpertLayer::quantizeFp8(hip, bytes.first(8), E, H, I); }, "short payload");
    expectInvalid([&] { (void)DeviceExpertLayer::quantizeFp8(hip, bytes, E, H, 0); }, "no columns");
    const auto layer = DeviceExpertLayer::quantizeFp8(hip, bytes, E, H, I);
    expect(layer->dtype() == DType::FP8 && layer->experts() == E && layer->hidden() == H &&
               layer->intermediate() == I, "the layer's description");
    const auto& d = layer->descriptor();
    std::vector<unsigned char> q(E * (2 * I * 256 + H * 256));
    std::vector<float> s(E * 3 * 4);
    hip->copyFromDevice(q.data(), d.packed, q.size());
    hip->copyFromDevice(s.data(), d.scale, s.size() * 4);

    // every byte and scale, and the payload that they stand for
    std::vector<float> back(p.size());
    std::size_t wrong = 0, at = 0;
    for (std::size_t e = 0; e < E; ++e) {
        for (std::size_t j = 0; j < 3; ++j) {
            const std::size_t K = j < 2 ? H : I, N = j < 2 ? I : H;
            const float* src = p.data() + (e * 3 + j) * H * I;
            float* dst = back.data() + (e * 3 + j) * H * I;
            const float* sc = s.data() + (e * 3 + j) * 4;
            for (std::size_t nb = 0; nb < 2; ++nb) {
                for (std::size_t kb = 0; kb < 2; ++kb) {
                    double amax = std::ldexp(1.0, -100);
                    for (std::size_t n = 128 * nb; n < std::min(N, 128 * nb + 128); ++n)
                        for (std::size_t k = 128 * kb; k < std::min(K, 128 * kb + 128); ++k)
                            amax = std::max(amax, (double)std::fabs(src[k * N + n]));
                    wrong += sc[nb * 2 + kb] != (float)(amax / 448.0);
                    for (std::size_t n = 128 * nb; n < std::min(N, 128 * nb + 128); ++n) {
                        for (std::size_t k = 128 * kb; k < 128 * kb + 128; ++k) {
                            const unsigned got = q[at + n * 256 + k];
                            wrong += got != (k < K ? nearest(src[k * N + n] * 448.0 / amax) : 0u);
                            if (k < K) dst[k * N + n] = (float)(e4m3(got) * sc[nb * 2 + kb]);
                        }
                    }
                }
            }
            at += N * 256;
        }
    }
    expect(wrong == 0, std::to_string(wrong) + " bytes or scales differ from the definition");

    // A block on it against the oracle on the values that the bytes stand for.  What is left is the
    // rounding of x and z to e4m3, half a step of at most 2^-3 each: in gate and up (silu's slope is at
    // most 1.1) and down, three times 2^-4 of the sums' absolute values, and 0.1 normwise with signs mixed.
    const std::size_t T = 21, k = 2;
    std::vector<float> h(T * H), w(H * E), out(T * H), ref(T * H), scores(T * k);
    std::vector<std::uint32_t> ids(T * k);
    hm_synth_normal(5, 2, (int64_t)h.size(), 0.0F, 1.0F, h.data());
    hm_synth_normal(5, 3, (int64_t)w.size(), 0.0F, 0.2F, w.data());
    tensor::HipTensorBackend tb(hip);
    auto dh = tb.allocateTensor(Shape{T, H}, DType::FP32);
    auto dw = tb.allocateTensor(Shape{H, E}, DType::FP32);
    hip->copyToDevice(dh.data(), h.data(), h.size() * 4);
    hip->copyToDevice(dw.data(), w.data(), w.size() * 4);
    HipMoEBlock block(hip, {E, k, router::RoutingNormalization::Softmax, true});
    block.addLayer(2, layer);
    auto res = block.executeBatch(2, dh.view(), dw.view());
    hip->copyFromDevice(out.data(), res.output.data(), out.size() * 4);
    hmo_layer ol{(int64_t)E, (int64_t)H, (int64_t)I, 0, back.data(), nullptr, nullptr};
    hmo_moe_block(&ol, h.data(), w.data(), (int64_t)T, (int32_t)k, 1, 1, ref.data(), ids.data(),
                  scores.data());
    bool routed = res.routing.tokens.size() == T;
    for (std::size_t t = 0; t < T && routed; ++t)
        for (std::size_t r = 0; r < k; ++r)
            routed &= res.routing.tokens[t].selectedExpertIds[r] == ids[t * k + r];
    expect(routed, "routing as the oracle's");
    double diff = 0.0, norm = 0.0;
    for (std::size_t i = 0; i < out.size(); ++i) {
        diff += ((double)out[i] - ref[i]) * ((double)out[i] - ref[i]);
        norm += (double)ref[i] * ref[i];
    }
    expect(norm > 0.0 && std::sqrt(diff / norm) <= 0.1, "block output " + std::to_string(std::sqrt(diff / norm)) +
                                                            " off the oracle's");
}

}  // namespace

int main(int argc, char** argv) {
    const std::string mode = argc > 1 ? argv[1] : "cpu";
    try {
        if (mode == "cpu") {
            cpuTests();
        } else if (mode == "gpu") {
            auto hip = std::make_shared<backend::HipBackend>(0);
            expect(hip->isAvailable(), "a HIP device is available");
            if (hip->isAvailable()) gpuTests(hip);
        } else {
            std::fprintf(stderr, "usage: test_fp8 cpu|gpu\n");
            return 2;
        }
    } catch (const std::exception& e) {
        std::fprintf(stderr, "FAIL: uncaught exception: %s\n", e.what());
        ++g_failures;
    }
    std::printf("%s: %d checks, %d failures\n", mode.c_str(), g_checks, g_failures);
    return g_failures == 0 ? 0 : 1;
}
