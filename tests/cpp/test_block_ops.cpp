// The block operators of the C++ interface, run in the order in which a transformer block has them, against loops in double
// precision: norm_residual_fwd -> rope_packed -> attention_window_fwd_packed -> attention_window_bwd_packed -> rope_packed
// (inverse) -> norm_residual_bwd, and attention_window_decode over the last token.  Each step is checked from what the step
// before left on the device.  Plain main(), exit code 0 = all checks passed.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include "llmt/core/arena.h"
#include "llmt/core/device.h"
#include "llmt/core/error.h"
#include "llmt/kernels/attention.h"
#include "llmt/kernels/norm_residual.h"
#include "llmt/kernels/rope.h"
#include "llmt_b200.h"

using namespace llmt;

namespace {

using Values = std::vector<double>;
int g_checks = 0, g_failures = 0;

uint16_t to_bf16(double x) {
    const float f = static_cast<float>(x);
    uint32_t u;
    std::memcpy(&u, &f, 4);
    return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
double of_bf16(uint16_t h) {
    const uint32_t u = static_cast<uint32_t>(h) << 16;
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}

uint64_t g_state = 1;
double uniform() {  // -1 .. 1
    g_state = g_state * 6364136223846793005ull + 1442695040888963407ull;
    return static_cast<double>(g_state >> 11) * 0x1p-52 - 1.0;
}

Tensor upload(Arena& arena, const Shape& shape, DType dtype, const Values& v) {
    Tensor t = arena.alloc(shape, dtype);
    std::vector<char> raw(t.bytes());
    for (size_t i = 0; i < v.size(); ++i) {
        if (dtype == DType::BF16) reinterpret_cast<uint16_t*>(raw.data())[i] = to_bf16(v[i]);
        else if (dtype == DType::FP32) reinterpret_cast<float*>(raw.data())[i] = static_cast<float>(v[i]);
        else reinterpret_cast<int32_t*>(raw.data())[i] = static_cast<int32_t>(v[i]);
    }
    CUDA_CHECK(cudaMemcpy(t.data, raw.data(), raw.size(), cudaMemcpyHostToDevice));
    return t;
}
Tensor random_tensor(Arena& arena, const Shape& shape, DType dtype, double centre = 0.0) {
    Values v(static_cast<size_t>(shape.numel()));
    for (double& x : v) x = centre + uniform();
    return upload(arena, shape, dtype, v);
}
Values download(const Tensor& t) {
    std::vector<char> raw(t.bytes());
    CUDA_CHECK(cudaMemcpy(raw.data(), t.data, raw.size(), cudaMemcpyDeviceToHost));
    Values v(static_cast<size_t>(t.numel()));
    for (size_t i = 0; i < v.size(); ++i)
        v[i] = t.dtype == DType::BF16 ? of_bf16(reinterpret_cast<uint16_t*>(raw.data())[i]) : reinterpret_cast<float*>(raw.data())[i];
    return v;
}

// |got - want| <= rtol |want| + atol for every element.
void check(const char* what, const Values& got, const Values& want, double rtol, double atol) {
    ++g_checks;
    for (size_t i = 0; i < want.size(); ++i)
        if (got.size() != want.size() || !(std::fabs(got[i] - want[i]) <= rtol * std::fabs(want[i]) + atol)) {
            ++g_failures;
            std::fprintf(stderr, "FAIL %s: [%zu] got %.9g want %.9g\n", what, i, got[i], want[i]);
            return;
        }
    std::printf("ok   %s\n", what);
}

constexpr int64_t B = 2, T = 37, H = 4, HKV = 2, HD = 32, ROT = 16, W = (H + 2 * HKV) * HD, C = 72, WINDOW = 11, SINKS = 2;
constexpr double kBf16 = 0x1p-8;  // half a step, relative

bool sees(int64_t i, int64_t j) { return j <= i && (j > i - WINDOW || j < SINKS); }

Values turned(const Values& qkv, const std::vector<double>& freqs, int64_t offset, bool inverse) {
    Values r = qkv;
    for (int64_t b = 0; b < B; ++b)
        for (int64_t t = 0; t < T; ++t)
            for (int64_t h = 0; h < H + HKV; ++h)
                for (int64_t i = 0; i < ROT / 2; ++i) {
                    const size_t at = static_cast<size_t>((b * T + t) * W + h * HD + i);
                    const double a = static_cast<double>(t + offset) * freqs[static_cast<size_t>(i)] * (inverse ? -1 : 1), u = qkv[at], w = qkv[at + ROT / 2];
                    r[at] = u * std::cos(a) - w * std::sin(a);
                    r[at + ROT / 2] = u * std::sin(a) + w * std::cos(a);
                }
    return r;
}

}  // namespace

int main() {
    Device dev(0);
    const RunCtx ctx = dev.make_ctx(0, KernelBackend::Naive, PrecisionPolicy::bf16_mixed());
    Arena arena(16 << 20, "block-ops-test");
    const int64_t rows = B * T;

    // ---- norms around the block: x fp32, y and h bf16, a gate per sequence
    const Tensor x = random_tensor(arena, {B, T, C}, DType::FP32), y = random_tensor(arena, {B, T, C}, DType::BF16);
    const Tensor w_post = random_tensor(arena, {C}, DType::FP32, 1.0), w_pre = random_tensor(arena, {C}, DType::FP32, 1.0),
                 gate = random_tensor(arena, {B, C}, DType::FP32);
    Tensor out = arena.alloc({B, T, C}, DType::FP32), h = arena.alloc({B, T, C}, DType::BF16);
    Tensor rstd_post = arena.alloc({rows}, DType::FP32), rstd_pre = arena.alloc({rows}, DType::FP32);
    kernels::NormResidual n;
    n.w_post = &w_post; n.gate = &gate; n.w_pre = &w_pre; n.rstd_post = &rstd_post; n.rstd_pre = &rstd_pre;
    n.scale = 0.5f;
    kernels::norm_residual_fwd(ctx, &out, &h, x, &y, n);
    dev.synchronize();
    const Values vx = download(x), vy = download(y), wp = download(w_post), wq = download(w_pre), vg = download(gate);
    Values want_out(vx.size()), want_h(vx.size()), rp(static_cast<size_t>(rows)), rq(static_cast<size_t>(rows));
    for (int64_t r = 0; r < rows; ++r) {
        double s = 0, q = 0;
        for (int64_t c = 0; c < C; ++c) s += vy[static_cast<size_t>(r * C + c)] * vy[static_cast<size_t>(r * C + c)];
        const double a = 1 / std::sqrt(s / C + static_cast<double>(n.eps));
        for (int64_t c = 0; c < C; ++c) {
            const size_t i = static_cast<size_t>(r * C + c);
            want_out[i] = vx[i] + 0.5 * vg[static_cast<size_t>(r / T * C + c)] * vy[i] * a * wp[static_cast<size_t>(c)];
            q += want_out[i] * want_out[i];
        }
        rp[static_cast<size_t>(r)] = a;
        rq[static_cast<size_t>(r)] = 1 / std::sqrt(q / C + static_cast<double>(n.eps));
        for (int64_t c = 0; c < C; ++c) want_h[static_cast<size_t>(r * C + c)] = want_out[static_cast<size_t>(r * C + c)] * rq[static_cast<size_t>(r)] * wq[static_cast<size_t>(c)];
    }
    // fp32 sums of 72 values: a few 2^-24 each way; values up to 8, so 1e-5 covers some tens of roundings
    check("norm_residual_fwd out", download(out), want_out, 1e-5, 1e-5);
    check("norm_residual_fwd h", download(h), want_h, kBf16 * 1.01, 1e-5);
    check("norm_residual_fwd rstd_post", download(rstd_post), rp, 1e-5, 0);
    check("norm_residual_fwd rstd_pre", download(rstd_pre), rq, 1e-5, 0);

    // ---- rotary positions in the packed projection
    std::vector<double> freqs(ROT / 2);
    if (llmt_b200_rope_frequencies(freqs.data(), ROT, 10000.0, 1.0, 1.0, 32.0, 0.0) != LLMT_B200_OK) return 2;
    double* dfreqs = static_cast<double*>(arena.alloc_bytes(sizeof(double) * ROT / 2));
    CUDA_CHECK(cudaMemcpy(dfreqs, freqs.data(), sizeof(double) * ROT / 2, cudaMemcpyHostToDevice));
    Tensor qkv = random_tensor(arena, {B, T, W}, DType::BF16);
    Values before = download(qkv);
    kernels::RopeSpec rope;
    rope.freqs = dfreqs; rope.rot_dim = ROT; rope.offset = 1000;
    kernels::rope_packed(ctx, qkv, H, HKV, rope);
    dev.synchronize();
    check("rope_packed", download(qkv), turned(before, freqs, 1000, false), kBf16 * 1.01, 1e-5);

    // ---- attention, forward and backward
    Tensor att = arena.alloc({B, T, H * HD}, DType::BF16), lse = arena.alloc({B, H, T}, DType::FP32);
    kernels::WindowSpec win;
    win.window = WINDOW; win.sinks = SINKS;
    kernels::attention_window_fwd_packed(ctx, att, &lse, qkv, H, HKV, win);
    dev.synchronize();
    const Values p = download(qkv), vatt = download(att);
    auto at = [&](const Values& v, int64_t b, int64_t t, int64_t head, int64_t d) { return v[static_cast<size_t>((b * T + t) * W + head * HD + d)]; };
    const double scale = 1 / std::sqrt(static_cast<double>(HD));
    std::vector<double> probs(static_cast<size_t>(B * H * T * T), 0.0);
    Values want_att(vatt.size(), 0.0), want_lse(static_cast<size_t>(B * H * T));
    for (int64_t b = 0; b < B; ++b)
        for (int64_t hh = 0; hh < H; ++hh)
            for (int64_t i = 0; i < T; ++i) {
                double sum = 0;
                double* row = &probs[static_cast<size_t>(((b * H + hh) * T + i) * T)];
                for (int64_t j = 0; j < T; ++j) {
                    if (!sees(i, j)) continue;
                    double s = 0;
                    for (int64_t d = 0; d < HD; ++d) s += at(p, b, i, hh, d) * at(p, b, j, H + hh / (H / HKV), d);
                    row[j] = std::exp(s * scale);  // |s scale| < 32 / sqrt(32) * 2: no overflow
                    sum += row[j];
                }
                want_lse[static_cast<size_t>((b * H + hh) * T + i)] = std::log(sum);
                for (int64_t j = 0; j < T; ++j) {
                    row[j] /= sum;
                    for (int64_t d = 0; d < HD; ++d)
                        want_att[static_cast<size_t>((b * T + i) * H * HD + hh * HD + d)] += row[j] * at(p, b, j, H + HKV + hh / (H / HKV), d);
                }
            }
    // P and the result are rounded once each: half a step of values up to sqrt(2), and of the result itself
    check("attention_window_fwd_packed y", vatt, want_att, kBf16 * 1.01, 1.5 * kBf16);
    check("attention_window_fwd_packed lse", download(lse), want_lse, 1e-5, 1e-5);

    Tensor dqkv = arena.alloc({B, T, W}, DType::BF16);
    const Tensor datt = random_tensor(arena, {B, T, H * HD}, DType::BF16);
    if (kernels::attention_window_workspace_bytes(qkv, H, HKV, win) > ctx.blas_workspace_bytes) return 2;
    kernels::attention_window_bwd_packed(ctx, dqkv, datt, qkv, att, lse, H, HKV, win);
    dev.synchronize();
    const Values da = download(datt);
    Values want_d(p.size(), 0.0), mass(p.size(), 0.0);  // mass: the same sums of absolute values
    for (int64_t b = 0; b < B; ++b)
        for (int64_t hh = 0; hh < H; ++hh)
            for (int64_t i = 0; i < T; ++i) {
                const int64_t hk = H + hh / (H / HKV), hv = hk + HKV;
                const double* row = &probs[static_cast<size_t>(((b * H + hh) * T + i) * T)];
                double dp[T], dsum = 0;
                for (int64_t j = 0; j < T; ++j) {
                    dp[j] = 0;
                    for (int64_t d = 0; d < HD; ++d) dp[j] += da[static_cast<size_t>((b * T + i) * H * HD + hh * HD + d)] * at(p, b, j, hv, d);
                    dsum += row[j] * dp[j];
                }
                for (int64_t j = 0; j < T; ++j)
                    for (int64_t d = 0; d < HD; ++d) {
                        const double ds = scale * row[j] * (dp[j] - dsum), bound = scale * row[j] * (std::fabs(dp[j]) + std::fabs(dsum) + 8),
                                     g = da[static_cast<size_t>((b * T + i) * H * HD + hh * HD + d)];
                        const size_t iq = static_cast<size_t>((b * T + i) * W + hh * HD + d), ik = static_cast<size_t>((b * T + j) * W + hk * HD + d),
                                     iv = static_cast<size_t>((b * T + j) * W + hv * HD + d);
                        want_d[iq] += ds * at(p, b, j, hk, d); mass[iq] += bound * std::fabs(at(p, b, j, hk, d));
                        want_d[ik] += ds * at(p, b, i, hh, d); mass[ik] += bound * std::fabs(at(p, b, i, hh, d));
                        want_d[iv] += row[j] * g; mass[iv] += row[j] * std::fabs(g);
                    }
            }
    // Every term carries a rounding of P or dS (and D one of `out`, whose dot with dO is up to 8 values' half steps: the 8
    // in `bound`), the result one more.
    {
        ++g_checks;
        const Values got = download(dqkv);
        bool ok = true;
        for (size_t i = 0; i < got.size() && ok; ++i) {
            ok = std::fabs(got[i] - want_d[i]) <= kBf16 * 1.01 * (std::fabs(want_d[i]) + mass[i]) + 1e-5;
            if (!ok) std::fprintf(stderr, "FAIL attention_window_bwd_packed: [%zu] got %.9g want %.9g (mass %.3g)\n", i, got[i], want_d[i], mass[i]);
        }
        if (ok) std::printf("ok   attention_window_bwd_packed\n");
        else ++g_failures;
    }
    before = download(dqkv);
    kernels::rope_packed(ctx, dqkv, H, HKV, rope, true);
    dev.synchronize();
    check("rope_packed inverse", download(dqkv), turned(before, freqs, 1000, true), kBf16 * 1.01, 1e-5);

    // ---- the last token over a cache that holds T of T + 3 places
    {
        Values ck(static_cast<size_t>(B * (T + 3) * HKV * HD), NAN), cv = ck, q1(static_cast<size_t>(B * W)), want(static_cast<size_t>(B * H * HD));
        for (int64_t b = 0; b < B; ++b) {
            for (int64_t t = 0; t < T; ++t)
                for (int64_t e = 0; e < HKV * HD; ++e) {
                    ck[static_cast<size_t>((b * (T + 3) + t) * HKV * HD + e)] = at(p, b, t, H, e);
                    cv[static_cast<size_t>((b * (T + 3) + t) * HKV * HD + e)] = at(p, b, t, H + HKV, e);
                }
            for (int64_t e = 0; e < W; ++e) q1[static_cast<size_t>(b * W + e)] = at(p, b, T - 1, 0, e);
            for (int64_t e = 0; e < H * HD; ++e) want[static_cast<size_t>(b * H * HD + e)] = want_att[static_cast<size_t>((b * T + T - 1) * H * HD + e)];
        }
        const Tensor q = upload(arena, {B, W}, DType::BF16, q1), k = upload(arena, {B, T + 3, HKV, HD}, DType::BF16, ck),
                     v = upload(arena, {B, T + 3, HKV, HD}, DType::BF16, cv), lengths = upload(arena, {B}, DType::I32, {T, T});
        Tensor y1 = arena.alloc({B, H * HD}, DType::BF16);
        if (kernels::attention_window_decode_workspace_bytes(q, k, H, win) > ctx.blas_workspace_bytes) return 2;
        kernels::attention_window_decode(ctx, y1, q, k, v, &lengths, H, win);
        dev.synchronize();
        check("attention_window_decode", download(y1), want, kBf16 * 1.01, 1.5 * kBf16);
    }

    // ---- the norms' gradients, added to what is there (beta 1)
    const Tensor dout = random_tensor(arena, {B, T, C}, DType::FP32), dh = random_tensor(arena, {B, T, C}, DType::BF16);
    Tensor dx = arena.alloc({B, T, C}, DType::FP32), dy = arena.alloc({B, T, C}, DType::BF16);
    Tensor dw_post = random_tensor(arena, {C}, DType::FP32), dw_pre = random_tensor(arena, {C}, DType::FP32), dgate = random_tensor(arena, {B, C}, DType::FP32);
    Values want_wp = download(dw_post), want_wq = download(dw_pre), want_g = download(dgate), want_dx(vx.size()), want_dy(vx.size());
    kernels::NormResidualGrads grads;
    grads.dw_post = &dw_post; grads.dgate = &dgate; grads.dw_pre = &dw_pre;
    if (kernels::norm_residual_workspace_bytes(dx, &y, n, grads) > ctx.blas_workspace_bytes) return 2;
    kernels::norm_residual_bwd(ctx, dx, &dy, &dout, &dh, &out, &y, n, grads);
    dev.synchronize();
    const Values vout = download(out), vdo = download(dout), vdh = download(dh);
    for (int64_t r = 0; r < rows; ++r) {
        double m = 0, e = 0;
        const double a = rp[static_cast<size_t>(r)], q = rq[static_cast<size_t>(r)];
        for (int64_t c = 0; c < C; ++c) m += vdh[static_cast<size_t>(r * C + c)] * wq[static_cast<size_t>(c)] * vout[static_cast<size_t>(r * C + c)] * q / C;
        for (int64_t c = 0; c < C; ++c) {
            const size_t i = static_cast<size_t>(r * C + c), ic = static_cast<size_t>(c), ig = static_cast<size_t>(r / T * C + c);
            want_dx[i] = vdo[i] + q * (vdh[i] * wq[ic] - vout[i] * q * m);
            e += 0.5 * vg[ig] * wp[ic] * want_dx[i] * vy[i] * a / C;
            want_wq[ic] += vdh[i] * vout[i] * q;
            want_wp[ic] += 0.5 * vg[ig] * want_dx[i] * vy[i] * a;
            want_g[ig] += 0.5 * wp[ic] * want_dx[i] * vy[i] * a;
        }
        for (int64_t c = 0; c < C; ++c) {
            const size_t i = static_cast<size_t>(r * C + c), ic = static_cast<size_t>(c), ig = static_cast<size_t>(r / T * C + c);
            want_dy[i] = a * (0.5 * vg[ig] * wp[ic] * want_dx[i] - vy[i] * a * e);
        }
    }
    // fp32 arithmetic on values of order 1, sums over 72 columns and 74 rows: some hundred roundings of 2^-24
    check("norm_residual_bwd dx", download(dx), want_dx, 1e-5, 2e-5);
    check("norm_residual_bwd dy", download(dy), want_dy, kBf16 * 1.01, 2e-5);
    check("norm_residual_bwd dw_post", download(dw_post), want_wp, 1e-5, 1e-4);
    check("norm_residual_bwd dgate", download(dgate), want_g, 1e-5, 1e-4);
    check("norm_residual_bwd dw_pre", download(dw_pre), want_wq, 1e-5, 1e-4);

    std::printf("%d checks, %d failures\n", g_checks, g_failures);
    return g_failures == 0 ? 0 : 1;
}
