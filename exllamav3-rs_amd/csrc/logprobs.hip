// Log probabilities, entropy and top alternatives of logits rows for gfx950: exl3r_token_logprobs.
//
// With m the row's maximum, l = sum_c e^(x_c - m) and t = sum_c e^(x_c - m) (x_c - m):
//   ln P_c = x_c - m - ln l,    entropy = ln l - t / l   (two terms >= 0: nothing cancels).
// A row is cut into slices of a workgroup each; a slice keeps its running m, l, t and the maximum of every group
// of 64 columns.  A second kernel, a workgroup per row, joins the slices and finds the top columns: with (value, lower
// column first) as the order, the k largest columns are in the k groups with the largest (maximum, lower group
// first), since each of those k groups has a column that precedes all columns of any other group.  Only these
// groups are read again.
#include "abi.hpp"
#include "common.cuh"

namespace exl3r {

constexpr int kLpGroup = 64;      // columns per group
constexpr int kLpMaxTop = 32;

struct LpArgs
{
    const char* x;
    int64_t ld;               // bytes
    int64_t n, vocab, rows;
    const int64_t* tokens;
    float* logprobs;
    float* entropy;
    int64_t* top_ids;
    float* top_logprobs;
    int32_t* err;
    float* part;              // [rows][slices][3]: m, l, t
    float* gmax;              // [rows][groups]
    int64_t groups;
    int32_t slices, top, dtype;
};

__device__ __forceinline__ float lp_max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Order-preserving 32-bit image of a float; -0 maps with +0 and every NaN to the top.
__device__ __forceinline__ uint32_t lp_order(float v)
{
    if (v != v) return 0xffffffffu;
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// Larger value, then lower index; below ~0 for every value and index, above 0.
__device__ __forceinline__ uint64_t lp_key(float v, uint32_t i) { return ((uint64_t)lp_order(v) << 32) | (0xfffffffeu - i); }
__device__ __forceinline__ uint32_t lp_index(uint64_t k) { return 0xfffffffeu - (uint32_t)k; }

__device__ __forceinline__ uint64_t lp_block_max(uint64_t v, uint64_t* lds)
{
    #pragma unroll
    for (int d = 1; d < 64; d <<= 1)
    {
        const uint64_t o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) v = lds[w] > v ? lds[w] : v;
    return v;
}

struct LpSum
{
    float m = -INFINITY, l = 0.0f, t = 0.0f;

    // A -inf logit adds nothing (its x - m is kept finite for the product with its zero weight); a NaN or +inf
    // makes l NaN.
    __device__ __forceinline__ void add8(const float (&x)[8], float cm)
    {
        const float mn = fmaxf(m, cm), ref = mn == -INFINITY ? 0.0f : mn;
        const float d = fmaxf(m - ref, -1e30f), r = __builtin_amdgcn_exp2f(d * kLog2e);
        t = r * fmaf(d, l, t);
        l *= r;
        #pragma unroll
        for (int j = 0; j < 8; ++j)
        {
            const float u = x[j] - ref, e = __builtin_amdgcn_exp2f(u * kLog2e);
            l += e;
            t = fmaf(e, fmaxf(u, -1e30f), t);
        }
        m = mn;
    }
    __device__ __forceinline__ void join(float m2, float l2, float t2)
    {
        const float mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.0f : mn;
        const float d1 = fmaxf(m - ref, -1e30f), d2 = fmaxf(m2 - ref, -1e30f);
        const float r1 = __builtin_amdgcn_exp2f(d1 * kLog2e), r2 = __builtin_amdgcn_exp2f(d2 * kLog2e);
        t = r1 * fmaf(d1, l, t) + r2 * fmaf(d2, l2, t2);
        l = r1 * l + r2 * l2;
        m = mn;
    }
};

// 256 lanes, 8 columns per lane and step: a group of 64 columns is 8 lanes of one step.
template <class IT>
__global__ __launch_bounds__(256) void k_lp_slices(LpArgs a, int64_t slice)
{
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / (uint32_t)a.slices, sl = blockIdx.x % (uint32_t)a.slices;
    const char* base = a.x + row * a.ld;
    const int64_t end = min(a.n, (sl + 1) * slice);
    LpSum s;
    for (int64_t c = sl * slice + tid * 8; c < ((end + 63) & ~(int64_t)63); c += 2048)
    {
        float x[8];
        #pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = c + j < end ? load1(base, IT::code, c + j) : -INFINITY;
        float cm = x[0];
        #pragma unroll
        for (int j = 1; j < 8; ++j) cm = lp_max_nan(cm, x[j]);
        s.add8(x, cm != cm ? -INFINITY : cm);
        float gm = cm;
        #pragma unroll
        for (int d = 1; d < 8; d <<= 1) gm = lp_max_nan(gm, __shfl_xor(gm, d));
        if ((tid & 7) == 0 && a.top) a.gmax[row * a.groups + c / kLpGroup] = gm;
    }
    #pragma unroll
    for (int d = 1; d < 64; d <<= 1)
    {
        const float m2 = __shfl_xor(s.m, d), l2 = __shfl_xor(s.l, d), t2 = __shfl_xor(s.t, d);
        s.join(m2, l2, t2);
    }
    __shared__ float w[4][3];
    if ((tid & 63) == 0) { w[tid >> 6][0] = s.m; w[tid >> 6][1] = s.l; w[tid >> 6][2] = s.t; }
    __syncthreads();
    if (tid == 0)
    {
        for (int i = 1; i < 4; ++i) s.join(w[i][0], w[i][1], w[i][2]);
        float* p = a.part + 3 * (row * a.slices + sl);
        p[0] = s.m; p[1] = s.l; p[2] = s.t;
    }
}

template <class IT>
__global__ __launch_bounds__(256) void k_lp_rows(LpArgs a)
{
    __shared__ uint64_t red[4];
    __shared__ uint32_t chosen[kLpMaxTop];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const char* base = a.x + row * a.ld;
    const float* part = a.part + 3 * row * a.slices;
    float m = -INFINITY;
    for (int i = 0; i < a.slices; ++i) m = fmaxf(m, part[3 * i]);
    double l = 0.0, t = 0.0;
    for (int i = 0; i < a.slices; ++i)
    {
        const float li = part[3 * i + 1];
        if (li == 0.0f) continue;
        const double d = (double)part[3 * i] - m, r = exp(d);
        l += r * li;
        t += r * (part[3 * i + 2] + d * li);
    }
    // ln P = (x - m) - ln l: m + ln l would lose ln l beside a large m.  Nothing but -inf: no distribution.
    const double ll = l == 0.0 ? (double)NAN : log(l);
    const auto log_p = [&](int64_t c) { return (float)((double)load1(base, IT::code, c) - m - ll); };
    if (tid == 0)
    {
        if (a.tokens)
        {
            const int64_t k = a.tokens[row];
            if (a.err && (k < 0 || k >= a.vocab)) *a.err = 1;
            a.logprobs[row] = k < 0 || k >= a.n ? (ll != ll ? NAN : -INFINITY) : log_p(k);
        }
        if (a.entropy) a.entropy[row] = (float)(ll - t / l);
    }
    const int top = a.top, ng = (int)min((int64_t)top, a.groups);
    uint64_t last = ~0ull;
    for (int i = 0; i < ng; ++i)
    {
        uint64_t best = 0;
        for (int64_t g = tid; g < a.groups; g += 256)
        {
            const uint64_t k = lp_key(a.gmax[row * a.groups + g], (uint32_t)g);
            if (k < last && k > best) best = k;
        }
        last = lp_block_max(best, red);
        if (tid == 0) chosen[i] = lp_index(last);
    }
    __syncthreads();
    uint64_t keys[kLpMaxTop * kLpGroup / 256];
    #pragma unroll
    for (int i = 0; i < kLpMaxTop * kLpGroup / 256; ++i)
    {
        const int at = i * 256 + tid;
        keys[i] = 0;
        if (at < ng * kLpGroup)
        {
            const int64_t c = (int64_t)chosen[at / kLpGroup] * kLpGroup + at % kLpGroup;
            if (c < a.n) keys[i] = lp_key(load1(base, IT::code, c), (uint32_t)c);
        }
    }
    last = ~0ull;
    for (int r = 0; r < top; ++r)
    {
        uint64_t best = 0;
        #pragma unroll
        for (int i = 0; i < kLpMaxTop * kLpGroup / 256; ++i) best = keys[i] < last && keys[i] > best ? keys[i] : best;
        last = lp_block_max(best, red);
        if (tid == 0)
        {
            const int64_t c = lp_index(last);
            a.top_ids[row * top + r] = c;
            a.top_logprobs[row * top + r] = log_p(c);
        }
    }
}

}  // namespace exl3r

using namespace exl3r;

namespace {

struct LpPlan
{
    int64_t slice, slices, groups;
    size_t part_bytes, bytes;
};

LpPlan lp_plan(int64_t rows, int64_t vocab)
{
    LpPlan p;
    p.slice = 8192;
    while ((vocab + p.slice - 1) / p.slice > 256) p.slice *= 2;
    p.slices = (vocab + p.slice - 1) / p.slice;
    p.groups = (vocab + kLpGroup - 1) / kLpGroup;
    p.part_bytes = ((size_t)rows * p.slices * 12 + 255) & ~(size_t)255;
    p.bytes = p.part_bytes + (((size_t)rows * p.groups * 4 + 255) & ~(size_t)255);
    return p;
}

constexpr int64_t kLpMaxRows = 1 << 20, kLpMaxVocab = 1LL << 31;

}  // namespace

extern "C" size_t exl3r_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab)
{
    if (rows <= 0 || vocab <= 0 || rows > kLpMaxRows || vocab > kLpMaxVocab) return 0;
    return lp_plan(rows, vocab).bytes;
}

extern "C" int exl3r_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, int max_logit,
                                    const int64_t* tokens, float* logprobs, float* entropy, int top_k, int64_t* top_ids,
                                    float* top_logprobs, int32_t* err_flag, void* workspace, size_t workspace_bytes,
                                    void* stream)
{
    begin_call();
    const char* op = "exl3r_token_logprobs";
    if (!is_float_dtype(dtype)) return set_error(EXL3R_EDTYPE, "%s: unsupported logits dtype %s", op, dtype_name(dtype));
    if (rows < 0 || rows > kLpMaxRows || vocab <= 0 || vocab > kLpMaxVocab || (rows > 1 && ld < vocab))
        return set_error(EXL3R_EINVAL, "%s: invalid shape rows=%lld vocab=%lld ld=%lld", op, (long long)rows,
                         (long long)vocab, (long long)ld);
    const int64_t n = (max_logit <= 0 || max_logit > vocab) ? vocab : max_logit;
    if (top_k < 0 || top_k > kLpMaxTop || top_k > n)
        return set_error(EXL3R_EINVAL, "%s: top_k %d is not in 0..%lld", op, top_k, (long long)(n < kLpMaxTop ? n : kLpMaxTop));
    if (rows == 0) return EXL3R_OK;
    if (!logits || (tokens && !logprobs) || (top_k && (!top_ids || !top_logprobs)))
        return set_error(EXL3R_EINVAL, "%s: logits and the outputs asked for must be non-null", op);
    const LpPlan p = lp_plan(rows, n);
    if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < p.bytes)
        return set_error(EXL3R_EINVAL, "%s: the workspace must be 256-byte aligned and hold %zu bytes (%zu given)", op, p.bytes,
                         workspace ? workspace_bytes : 0);
    LpArgs a{};
    a.x = (const char*)logits;
    a.ld = (rows > 1 ? ld : vocab) * dtype_bytes(dtype);
    a.n = n; a.vocab = vocab; a.rows = rows;
    a.tokens = tokens; a.logprobs = logprobs; a.entropy = entropy;
    a.top_ids = top_ids; a.top_logprobs = top_logprobs; a.err = err_flag;
    a.part = (float*)workspace;
    a.gmax = (float*)((char*)workspace + p.part_bytes);
    a.groups = p.groups;
    a.slices = (int)p.slices;
    a.top = top_k;
    hipStream_t s = (hipStream_t)stream;
    if (rows * p.slices > 0xffffff) return set_error(EXL3R_EINVAL, "%s: more than 2^24 workgroups", op);
    with_float_type(dtype, [&](auto T) {
        using Ty = decltype(T);
        launch(k_lp_slices<Ty>, (unsigned)(rows * p.slices), 256, 0, s, a, p.slice);
        launch(k_lp_rows<Ty>, (unsigned)rows, 256, 0, s, a);
    });
    return launch_status(op);
}
