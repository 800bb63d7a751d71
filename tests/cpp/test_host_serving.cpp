// The host layer's serving calls: rope_paged_kv, paged_attn and paged_attn_shared in a row against sums in double over
// the cache that the first left, and token_logprobs.  `test_host_serving refusals` checks the arguments' checks, no GPU.
#include "exl3r.hpp"
#include "rowops_oracle.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <string>
#include <vector>

using namespace exl3r;

static int failures = 0;

static void report(const char* what, bool ok, double worst, double bound)
{
    std::printf("%s %s: worst %.3g of %.3g\n", ok ? "ok  " : "FAIL", what, worst, bound);
    failures += !ok;
}

static void refused(const char* what, int code, const std::function<void()>& f)
{
    try
    {
        f();
    }
    catch (const Error& e)
    {
        const bool ok = e.code() == code;
        std::printf("%s %s: %s\n", ok ? "ok  " : "FAIL", what, e.what());
        failures += !ok;
        return;
    }
    std::printf("FAIL %s: no exception\n", what);
    ++failures;
}

static void refusals()
{
    void* const fake = (void*)0x1000;
    Stream s;
    const Tensor q(fake, DType::F16, { 2, 3, 8, 128 }), kc(fake, DType::F16, { 8, 16, 2, 128 }), bt(fake, DType::I32, { 2, 4 });
    const Tensor sl(fake, DType::I32, { 2 });
    const auto attn = [&](const Tensor& q_, const Tensor& kc_, const Tensor& vc_, const Tensor& bt_, const Tensor& sl_,
                          const Tensor& out_, int window, int sinks, const Tensor* lse) {
        ffi::paged_attn(q_, kc_, vc_, bt_, sl_, out_, 0.0f, window, sinks, lse, nullptr, nullptr, s);
    };
    const Tensor kb(fake, DType::BF16, { 8, 16, 2, 128 }), k64(fake, DType::F16, { 8, 16, 2, 64 }), bt3(fake, DType::I32, { 3, 4 });
    const Tensor btl(fake, DType::I64, { 2, 4 }), lse2(fake, DType::F32, { 2, 3 }), q96(fake, DType::F16, { 2, 3, 8, 96 });
    const Tensor k96(fake, DType::F16, { 8, 16, 2, 96 }), k3(fake, DType::F16, { 8, 16, 3, 128 }), kp(fake, DType::F16, { 8, 12, 2, 128 });
    const Tensor gap(fake, DType::F16, { 2, 3, 8, 128 }, { 5000, 1024, 128, 1 });
    const Tensor qf(fake, DType::F32, { 2, 3, 8, 128 }), kf(fake, DType::F32, { 8, 16, 2, 128 });
    refused("paged_attn cache dtype", EXL3R_EINVAL, [&] { attn(q, kb, kb, bt, sl, q, 0, 0, nullptr); });
    refused("paged_attn cache head_dim", EXL3R_EINVAL, [&] { attn(q, k64, k64, bt, sl, q, 0, 0, nullptr); });
    refused("paged_attn table rows", EXL3R_EINVAL, [&] { attn(q, kc, kc, bt3, sl, q, 0, 0, nullptr); });
    refused("paged_attn table dtype", EXL3R_EINVAL, [&] { attn(q, kc, kc, btl, sl, q, 0, 0, nullptr); });
    refused("paged_attn lse shape", EXL3R_EINVAL, [&] { attn(q, kc, kc, bt, sl, q, 0, 0, &lse2); });
    refused("paged_attn batch stride", EXL3R_EINVAL, [&] { attn(gap, kc, kc, bt, sl, q, 0, 0, nullptr); });
    refused("paged_attn head_dim 96", EXL3R_EINVAL, [&] { attn(q96, k96, k96, bt, sl, q96, 0, 0, nullptr); });
    refused("paged_attn 8 heads on 3", EXL3R_EINVAL, [&] { attn(q, k3, k3, bt, sl, q, 0, 0, nullptr); });
    refused("paged_attn page size 12", EXL3R_EINVAL, [&] { attn(q, kp, kp, bt, sl, q, 0, 0, nullptr); });
    refused("paged_attn float32", EXL3R_EDTYPE, [&] { attn(qf, kf, kf, bt, sl, qf, 0, 0, nullptr); });
    refused("paged_attn sinks without a window", EXL3R_EINVAL, [&] { attn(q, kc, kc, bt, sl, q, 0, 4, nullptr); });
    refused("paged_attn_shared negative", EXL3R_EINVAL, [&] {
        ffi::paged_attn_shared(q, kc, kc, bt, sl, q, -16, 0.0f, 0, 0, nullptr, nullptr, nullptr, s);
    });
    refused("paged_attn_shared part of a page", EXL3R_EINVAL, [&] {
        ffi::paged_attn_shared(q, kc, kc, bt, sl, q, 8, 0.0f, 0, 0, nullptr, nullptr, nullptr, s);
    });
    refused("paged_attn_shared without its workspace", EXL3R_EINVAL, [&] {
        ffi::paged_attn_shared(q, kc, kc, bt, sl, q, 16, 0.0f, 0, 0, nullptr, nullptr, nullptr, s);
    });
    const Tensor l(fake, DType::F16, { 3, 1000 }), tok(fake, DType::I64, { 3 }), t32(fake, DType::I32, { 3 }), f(fake, DType::F32, { 3 });
    const Tensor ids(fake, DType::I64, { 3, 40 }), tl(fake, DType::F32, { 3, 40 }), tl2(fake, DType::F32, { 3, 20 }), f2(fake, DType::F32, { 2 });
    const auto lp = [&](const Tensor* t, const Tensor* o, const Tensor* e, const Tensor* i, const Tensor* v) {
        ffi::token_logprobs(l, t, o, e, i, v, 0, nullptr, nullptr, s);
    };
    refused("token_logprobs tokens alone", EXL3R_EINVAL, [&] { lp(&tok, nullptr, nullptr, nullptr, nullptr); });
    refused("token_logprobs int32 tokens", EXL3R_EINVAL, [&] { lp(&t32, &f, nullptr, nullptr, nullptr); });
    refused("token_logprobs short logprobs", EXL3R_EINVAL, [&] { lp(&tok, &f2, nullptr, nullptr, nullptr); });
    refused("token_logprobs ids alone", EXL3R_EINVAL, [&] { lp(nullptr, nullptr, nullptr, &ids, nullptr); });
    refused("token_logprobs unlike tops", EXL3R_EINVAL, [&] { lp(nullptr, nullptr, nullptr, &ids, &tl2); });
    refused("token_logprobs 40 tops", EXL3R_EINVAL, [&] { lp(nullptr, nullptr, nullptr, &ids, &tl); });
    refused("token_logprobs without its workspace", EXL3R_EINVAL, [&] { lp(&tok, &f, nullptr, nullptr, nullptr); });
}

static uint64_t seed = 20260101;
static double uniform()       // [-1, 1)
{
    seed = seed * 6364136223846793005ull + 1442695040888963407ull;
    return (double)(seed >> 11) * 0x1p-52 - 1.0;
}

static std::vector<uint16_t> halves(size_t n, double amp)
{
    std::vector<uint16_t> v(n);
    for (auto& x : v) x = oracle_f32_to_f16((float)(amp * uniform()));
    return v;
}

template <class T> static OwnedTensor upload(const std::vector<T>& h, DType dt, std::vector<int64_t> shape, const Stream& s)
{
    OwnedTensor t = OwnedTensor::empty(dt, shape);
    t.buf.upload(h.data(), h.size() * sizeof(T), s);
    return t;
}
template <class T> static std::vector<T> download(const OwnedTensor& t, const Stream& s)
{
    std::vector<T> h(t.buf.bytes() / sizeof(T));
    t.buf.download(h.data(), t.buf.bytes(), s);
    return h;
}

int main(int argc, char** argv)
{
    if (argc > 1 && std::string(argv[1]) == "refusals")
    {
        refusals();
        std::printf(failures ? "test_host_serving: %d failures\n" : "test_host_serving: all passed\n", failures);
        return failures != 0;
    }
    Stream s = Stream::create();
    // Two sequences on a shared first page of 16 keys and pages of their own, 19 and 37 cached positions.
    {
        const int bsz = 2, seq = 3, hq = 8, hk = 2, hd = 64, page = 16, pages = 8, blocks = 4;
        const std::vector<int32_t> table = { 5, 1, 6, 2, 5, 7, 3, 0 }, lens = { 19, 37 };
        auto kc = upload(halves((size_t)pages * page * hk * hd, 2.0), DType::F16, { pages, page, hk, hd }, s);
        auto vc = upload(halves((size_t)pages * page * hk * hd, 2.0), DType::F16, { pages, page, hk, hd }, s);
        auto q = upload(halves((size_t)bsz * seq * hq * hd, 2.0), DType::F16, { bsz, seq, hq, hd }, s);
        auto k = upload(halves((size_t)bsz * seq * hk * hd, 2.0), DType::F16, { bsz, seq, hk, hd }, s);
        auto v = upload(halves((size_t)bsz * seq * hk * hd, 2.0), DType::F16, { bsz, seq, hk, hd }, s);
        auto bt = upload(table, DType::I32, { bsz, blocks }, s), sl = upload(lens, DType::I32, { bsz }, s);
        const std::vector<float> inv = RoPE::default_inv_freq(1e4, hd);
        auto inv_t = upload(inv, DType::F32, { hd / 2 }, s);
        ffi::rope_paged_kv(q.t, q.t, k.t, nullptr, v.t, inv_t.t, 0, &sl.t, nullptr, nullptr, 1e-6f, 0.f, RopeStyle::NeoX, 1.f,
                           kc.t, vc.t, bt.t, sl.t, nullptr, s);
        const auto qh = download<uint16_t>(q, s), kh = download<uint16_t>(kc, s), vh = download<uint16_t>(vc, s);
        auto out = OwnedTensor::empty(DType::F16, { bsz, seq, hq, hd }), lse = OwnedTensor::empty(DType::F32, { bsz, seq, hq });
        for (int shared = 0; shared <= page; shared += page)
            for (int window = 0; window <= 20; window += 20)
            {
                const size_t need = ffi::paged_attn_workspace_bytes(q.t, kc.t, bt.t, shared);
                DeviceBuffer ws(need ? need : 256);
                const int sinks = window ? 2 : 0;
                if (shared) ffi::paged_attn_shared(q.t, kc.t, vc.t, bt.t, sl.t, out.t, shared, 0.f, window, sinks, &lse.t, nullptr, &ws, s);
                else ffi::paged_attn(q.t, kc.t, vc.t, bt.t, sl.t, out.t, 0.f, window, sinks, &lse.t, nullptr, &ws, s);
                const auto oh = download<uint16_t>(out, s);
                const auto lh = download<float>(lse, s);
                double worst = 0.0, worst_lse = 0.0, vmax = 0.0;
                for (int b = 0; b < bsz; ++b)
                    for (int t = 0; t < seq; ++t)
                        for (int h = 0; h < hq; ++h)
                        {
                            const int p = lens[b] + t, kv = h / (hq / hk);
                            const size_t row = ((size_t)b * seq + t) * hq + h;
                            std::vector<double> sc, o(hd, 0.0);
                            std::vector<size_t> at;
                            double m = -INFINITY, l = 0.0;
                            for (int j = 0; j <= p; ++j)
                            {
                                if (window && p - j >= window && j >= sinks) continue;
                                const size_t r = ((size_t)(table[b * blocks + j / page] * page + j % page) * hk + kv) * hd;
                                double dot = 0.0;
                                for (int d = 0; d < hd; ++d) dot += (double)oracle_f16_to_f32(qh[row * hd + d]) * (double)oracle_f16_to_f32(kh[r + d]);
                                sc.push_back(dot / std::sqrt((double)hd));
                                at.push_back(r);
                                m = std::max(m, sc.back());
                            }
                            for (size_t i = 0; i < sc.size(); ++i)
                            {
                                const double e = std::exp(sc[i] - m);
                                l += e;
                                for (int d = 0; d < hd; ++d)
                                {
                                    const double x = (double)oracle_f16_to_f32(vh[at[i] + d]);
                                    o[d] += e * x;
                                    vmax = std::max(vmax, std::fabs(x));
                                }
                            }
                            for (int d = 0; d < hd; ++d) worst = std::max(worst, std::fabs((double)oracle_f16_to_f32(oh[row * hd + d]) - o[d] / l));
                            worst_lse = std::max(worst_lse, std::fabs(lh[row] - (m + std::log(l))));
                        }
                // Off by half a step where P and where the output are rounded to f16, 2^-11 each, and by the scores: 64
                // products in fp32, at most 8 a rotated pair, 64 * 2^-24 * 256 / 8 = 1.3e-4, which moves the weights by
                // less than 2 * 1.3e-4 < 2^-11.
                const double bound = 3.0 * 0x1p-11 * vmax;
                const std::string what = std::string(shared ? "paged_attn_shared" : "paged_attn") + (window ? ", window" : "");
                report(what.c_str(), worst <= bound, worst, bound);
                report((what + ": lse").c_str(), worst_lse <= 2e-4, worst_lse, 2e-4);
            }
    }
    // token_logprobs: f16 logits [5, 3001], every column and the first 2500.
    for (int limit = 0; limit <= 2500; limit += 2500)
    {
        const int rows = 5, vocab = 3001, top = 4, n = limit ? limit : vocab;
        const auto lh = halves((size_t)rows * vocab, 8.0);
        std::vector<int64_t> tok(rows);
        for (int r = 0; r < rows; ++r) tok[r] = 400 * r + 11;
        auto l = upload(lh, DType::F16, { rows, vocab }, s), t = upload(tok, DType::I64, { rows }, s);
        auto lp = OwnedTensor::empty(DType::F32, { rows }), ent = OwnedTensor::empty(DType::F32, { rows });
        auto ids = OwnedTensor::empty(DType::I64, { rows, top }), tl = OwnedTensor::empty(DType::F32, { rows, top });
        const size_t need = ffi::token_logprobs_workspace_bytes(l.t);
        DeviceBuffer ws(need ? need : 256);
        ffi::token_logprobs(l.t, &t.t, &lp.t, &ent.t, &ids.t, &tl.t, limit, nullptr, &ws, s);
        const auto gl = download<float>(lp, s), ge = download<float>(ent, s), gt = download<float>(tl, s);
        const auto gi = download<int64_t>(ids, s);
        double worst = 0.0;
        bool same = true;
        for (int r = 0; r < rows; ++r)
        {
            std::vector<double> x(n);
            for (int c = 0; c < n; ++c) x[c] = (double)oracle_f16_to_f32(lh[(size_t)r * vocab + c]);
            const double m = *std::max_element(x.begin(), x.end());
            double z = 0.0, u = 0.0;
            for (double v : x) { z += std::exp(v - m); u += std::exp(v - m) * (v - m); }
            worst = std::max({ worst, std::fabs(gl[r] - (x[tok[r]] - m - std::log(z))), std::fabs(ge[r] - (std::log(z) - u / z)) });
            std::vector<int64_t> order(n);
            for (int c = 0; c < n; ++c) order[c] = c;
            std::stable_sort(order.begin(), order.end(), [&](int64_t a, int64_t b) { return x[a] > x[b]; });
            for (int i = 0; i < top; ++i)
            {
                same = same && gi[r * top + i] == order[i];
                worst = std::max(worst, std::fabs(gt[r * top + i] - (x[order[i]] - m - std::log(z))));
            }
        }
        // Sums of 3001 terms in at most 32 + 16 additions each, 2^-24 a step, exponentials within 2^-22, the result
        // (below 32) rounded once: 48 * 2^-24 + 2^-22 + 16 * 2^-23 < 8e-6; the entropy's two terms, below 16, likewise.
        report("token_logprobs", worst <= 4e-5 && same, worst, 4e-5);
    }
    std::printf(failures ? "test_host_serving: %d failures\n" : "test_host_serving: all passed\n", failures);
    return failures != 0;
}
