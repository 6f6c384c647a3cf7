// expert_example.cpp -- an expert layer's products through the C++ Handle
// mirror (cublas_rs.hpp): tokens sorted by expert in 16 bits, with both
// gradients, and single tokens from 4-bit weights.
//
// Values are small whole numbers and scales powers of two, so every result is
// exact and is compared bit for bit with a sum on the host.  Exits 1 on the
// first difference.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "cublas_rs.hpp"

using namespace cublas_rs;

static void fail(const char *what) {
    std::fprintf(stderr, "FAIL: %s\n", what);
    std::exit(1);
}

template <typename F>
static void throws(const char *what, CublasError::Kind kind, F call) {
    try {
        call();
    } catch (const CublasError &e) {
        if (e.kind() == kind) return;
    }
    fail(what);
}

// Whole numbers from -3 to 3.
struct Draw {
    uint32_t s;
    int operator()() {
        s = s * 1664525u + 1013904223u;
        return static_cast<int>((s >> 16) % 7u) - 3;
    }
};

template <typename H>
static std::vector<H> whole(size_t n, uint32_t seed, std::vector<float> &values) {
    Draw d{seed};
    std::vector<H> v(n);
    values.resize(n);
    for (size_t i = 0; i < n; ++i) v[i] = H::from_f32(values[i] = float(d()));
    return v;
}

template <typename H>
static void grouped(const Handle &h, size_t n, size_t k) {
    const std::vector<int32_t> off = {2, 40, 40, 173, 180};  // an empty group, rows of none at both ends
    const size_t groups = off.size() - 1, rows = 190;
    std::vector<float> a, b, c;
    auto da = h.upload(whole<H>(rows * k, 1, a)), db = h.upload(whole<H>(groups * k * n, 2, b)),
         dc = h.upload(whole<H>(rows * n, 3, c)), dx = h.template zeroed<H>(rows * k);
    auto doff = h.upload(off);
    auto dw = h.template zeroed<float>(groups * k * n);
    auto dw16 = h.template zeroed<H>(groups * k * n);
    h.hgemm_grouped_wgrad(GemmConfig<float>{k, n, rows, 1.0f, 0.0f}, groups, da, dc, doff, dw);
    h.hgemm_grouped_wgrad(GemmConfig<float>{k, n, rows, 1.0f, 0.0f}, groups, da, dc, doff, dw16);
    h.hgemm_grouped(GemmConfig<float>{rows, k, n, 1.0f, 0.0f}, groups, dc, db, doff, dx, Transpose::Trans);
    h.hgemm_grouped(GemmConfig<float>{rows, n, k, 2.0f, -1.0f}, groups, da, db, doff, dc);
    h.synchronize();
    const auto gc = h.download(dc), gx = h.download(dx), gw16 = h.download(dw16);
    const auto gw = h.download(dw);
    for (size_t r = 0; r < rows; ++r) {
        size_t g = 0;
        while (g < groups && !(int32_t(r) >= off[g] && int32_t(r) < off[g + 1])) ++g;
        for (size_t j = 0; j < n; ++j) {
            float sum = 0.0f;
            for (size_t i = 0; g < groups && i < k; ++i) sum += a[r * k + i] * b[(g * k + i) * n + j];
            const float want = g < groups ? 2.0f * sum - c[r * n + j] : c[r * n + j];
            if (gc[r * n + j].bits != H::from_f32(want).bits) fail("hgemm_grouped");
        }
        for (size_t i = 0; i < k; ++i) {
            float sum = 0.0f;
            for (size_t j = 0; g < groups && j < n; ++j) sum += c[r * n + j] * b[(g * k + i) * n + j];
            if (gx[r * k + i].bits != H::from_f32(sum).bits) fail("hgemm_grouped, transposed");
        }
    }
    for (size_t g = 0; g < groups; ++g)
        for (size_t i = 0; i < k; ++i)
            for (size_t j = 0; j < n; ++j) {
                float sum = 0.0f;
                for (int32_t r = off[g]; r < off[g + 1]; ++r) sum += a[r * k + i] * c[r * n + j];
                if (gw[(g * k + i) * n + j] != sum) fail("hgemm_grouped_wgrad, float");
                if (gw16[(g * k + i) * n + j].bits != H::from_f32(sum).bits) fail("hgemm_grouped_wgrad");
            }
    std::printf("  grouped products and gradients, n = %zu, k = %zu OK\n", n, k);
}

template <typename H>
static void four_bits(const Handle &h, size_t n, bool with_zeros) {
    // every group has -7 and 7 (with zero points -4 and 11) among its values,
    // times a power of two: scales are powers of two and values come back exactly
    const size_t m = 50, experts = 3, group = 32, gs = (n + group - 1) / group;
    std::vector<H> w(experts * m * n);
    std::vector<float> wf(w.size());
    Draw d{5};
    for (size_t r = 0; r < experts * m; ++r)
        for (size_t j = 0; j < n; ++j) {
            const float scale = j / group % 2 ? 0.25f : 2.0f;
            const float v = j % group == 0 ? (with_zeros ? -4.0f : -7.0f) : j % group == 1 ? (with_zeros ? 11.0f : 7.0f) : float(d());
            w[r * n + j] = H::from_f32(wf[r * n + j] = v * scale);
        }
    auto dw = h.upload(w), scales = h.template zeroed<H>(experts * m * gs), back = h.template zeroed<H>(w.size());
    auto packed = h.template zeroed<uint8_t>(experts * m * ((n + 1) / 2)), zeros = h.template zeroed<uint8_t>(experts * m * gs);
    DeviceBuffer<uint8_t> *z = with_zeros ? &zeros : nullptr;
    h.quantize_w4(experts * m, n, group, dw, packed, scales, z);
    h.dequantize_w4(experts * m, n, group, packed, scales, z, back);
    const std::vector<int32_t> index = {2, 0, 0, 3, 1};
    std::vector<float> x;
    auto dx = h.upload(whole<H>(3 * n, 6, x));
    auto di = h.upload(index);
    auto y = h.template zeroed<H>(5 * m), y1 = h.template zeroed<H>(3 * m);
    h.hgemv_w4_grouped(experts, m, n, group, 0.5f, packed, scales, z, dx, di, 0.0f, y, index.size(), 2);
    h.hgemv_w4(m, n, group, 1.0f, packed, scales, z, dx, 0.0f, y1, 3);
    h.synchronize();
    const auto gb = h.download(back), gy = h.download(y), gy1 = h.download(y1);
    for (size_t i = 0; i < w.size(); ++i)
        if (gb[i].to_f32() != wf[i]) fail("quantize_w4 and back");
    auto product = [&](size_t e, size_t row, size_t v) {
        float sum = 0.0f;
        for (size_t j = 0; j < n; ++j) sum += wf[(e * m + row) * n + j] * x[v * n + j];
        return sum;
    };
    for (size_t row = 0; row < m; ++row) {
        for (size_t i = 0; i < index.size(); ++i) {
            const float want = index[i] < int32_t(experts) ? 0.5f * product(size_t(index[i]), row, i / 2) : 0.0f;
            if (gy[i * m + row].bits != H::from_f32(want).bits) fail("hgemv_w4_grouped");
        }
        for (size_t i = 0; i < 3; ++i)
            if (gy1[i * m + row].bits != H::from_f32(product(0, row, i)).bits) fail("hgemv_w4");
    }
    std::printf("  4-bit weights, n = %zu%s OK\n", n, with_zeros ? ", zero points" : "");
}

static void refusals(const Handle &h) {
    using Kind = CublasError::Kind;
    auto a = h.zeroed<f16>(64), b = h.zeroed<f16>(128), c = h.zeroed<f16>(64);
    auto off = h.zeroed<int32_t>(3), few = h.zeroed<int32_t>(2);
    GemmConfig<float> cfg{8, 8, 8, 1.0f, 0.0f};
    throws("short B", Kind::DimensionMismatch, [&] { h.hgemm_grouped(cfg, 2, a, a, off, c); });
    throws("short offsets", Kind::DimensionMismatch, [&] { h.hgemm_grouped(cfg, 2, a, b, few, c); });
    throws("short gradient", Kind::DimensionMismatch, [&] { h.hgemm_grouped_wgrad(cfg, 2, a, b, off, c); });
    auto packed = h.zeroed<uint8_t>(8 * 16), z = h.zeroed<uint8_t>(7);
    auto w = h.zeroed<f16>(8 * 32), s = h.zeroed<f16>(8);
    throws("short zeros", Kind::DimensionMismatch, [&] { h.quantize_w4(8, 32, 32, w, packed, s, &z); });
    throws("group of 0", Kind::InvalidArgument, [&] { h.quantize_w4(8, 32, 0, w, packed, s); });
    throws("fan of 0", Kind::InvalidArgument,
           [&] { h.hgemv_w4_grouped(1, 8, 32, 32, 1.0f, packed, s, nullptr, w, off, 0.0f, c, 2, 0); });
    throws("short x", Kind::DimensionMismatch,
           [&] { h.hgemv_w4_grouped(1, 8, 32, 32, 1.0f, packed, s, nullptr, s, off, 0.0f, c, 2, 2); });
    h.hgemm_grouped(GemmConfig<float>{0, 8, 8, 1.0f, 0.0f}, 2, a, b, off, c);  // no rows
    auto wrong = h.upload(std::vector<int32_t>{0, 9, 8});
    h.hgemm_grouped(cfg, 2, a, b, wrong, c);
    throws("offsets that do not ascend", Kind::InvalidArgument, [&] { h.synchronize(); });
    std::printf("  refusals OK\n");
}

int main() {
    try {
        for (float f : {1.0f, -2.5f, 1.00390625f, 1.01171875f, 3.0e38f, 1.0e-40f})  // ties to even
            if (std::fabs(bf16::from_f32(f).to_f32() - f) > std::fabs(f) / 256 + 1e-40f) fail("bf16");
        if (bf16::from_f32(1.00390625f).bits != 0x3f80 || bf16::from_f32(1.01171875f).bits != 0x3f82 ||
            !std::isnan(bf16::from_f32(NAN).to_f32()))
            fail("bf16 ties");
        Handle h = Handle::create();
        grouped<f16>(h, 72, 40);
        grouped<bf16>(h, 33, 65);
        for (bool with_zeros : {false, true}) {
            four_bits<f16>(h, 96, with_zeros);
            four_bits<bf16>(h, 67, with_zeros);
        }
        refusals(h);
    } catch (const CublasError &e) {
        std::fprintf(stderr, "CublasError: %s\n", e.what());
        return 1;
    }
    std::printf("all OK\n");
    return 0;
}
