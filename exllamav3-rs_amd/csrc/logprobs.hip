// Log probabilities, entropy and top alternatives of logits rows for gfx950: exl3r_token_logprobs.
//
// With m the row's maximum, l = sum_c e^(x_c - m) and t = sum_c e^(x_c - m) (x_c - m):
//   ln P_c = x_c - m - ln l,    entropy = ln l - t / l   (two terms >= 0: nothing cancels).
// Each lane keeps a running m, l, t over steps of 32 columns (4 chunks of 8, 2048 apart, so a wave's loads are whole
// lines), and the maximum of each of its steps: a group of 32 columns.  The top columns are then found from the group
// maxima alone.  A lane's best group maximum is one column's value, so with T the k-th largest of the lanes' best, k
// columns reach T at least, and every column among the k largest does: only the groups whose maximum reaches T, a few
// more than k, are read again, and their columns that reach T, as (value, lower column) keys, ranked by counting.
//
// Bound by reading the logits: 4096 rows of 151936 bf16 with 5 alternatives 203 us, 6.1 TB/s.  Few rows by latency: 64
// rows of 151936 fp32 with 20 alternatives 18 us (the slices 10, 3.9 TB/s, and 8 for a row's chain of loads, maxima,
// candidates and ranks), one row 11.6 us.
#include "abi.hpp"
#include "common.cuh"

namespace exl3r {

constexpr int kLpLanes = 256;
constexpr int kLpChunks = 4;                                 // chunks of 8 columns per lane and step
constexpr int kLpStep = kLpLanes * 8 * kLpChunks;            // columns per step of a workgroup
constexpr int kLpMaxTop = 32;
constexpr int kLpKeep = 24;                                  // group maxima per lane that stay in registers (196608 columns)
constexpr int kLpList = 64;                                  // groups read again at most in the usual way
// Columns ranked at most: in the careful way, those of fewer than kLpMaxTop groups and, of the columns that share the
// floor's value, fewer than kLpMaxTop and one round of the search.
constexpr int kLpCands = kLpMaxTop * 8 * kLpChunks + kLpMaxTop + kLpLanes;

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
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    return v != v ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
// Larger value, then lower index; below ~0 for every value and index, above 0.
__device__ __forceinline__ uint64_t lp_key(float v, uint32_t i) { return ((uint64_t)lp_order(v) << 32) | (0xfffffffeu - i); }
__device__ __forceinline__ uint32_t lp_index(uint64_t k) { return 0xfffffffeu - (uint32_t)k; }
__device__ __forceinline__ float lp_value(uint64_t k)
{
    const uint32_t u = (uint32_t)(k >> 32);
    if (u == 0xffffffffu) return NAN;
    return __builtin_bit_cast(float, (u & 0x80000000u) ? u ^ 0x80000000u : ~u);
}

struct LpSum
{
    float m = -INFINITY, l = 0.0f, t = 0.0f;

    // A -inf logit adds nothing (its x - m is kept finite for the product with its zero weight); a NaN or +inf
    // makes l NaN.  cm: the maximum of x, NaNs aside.
    template <int N>
    __device__ __forceinline__ void add(const float (&x)[N], float cm)
    {
        const float mn = fmaxf(m, cm), ref = mn == -INFINITY ? 0.0f : mn;
        const float d = fmaxf(m - ref, -1e30f), r = __builtin_amdgcn_exp2f(d * kLog2e);
        // four short sums, so that the long ones take one addition per step
        float ls[4] = {}, ts[4] = {};
        #pragma unroll
        for (int j = 0; j < N; ++j)
        {
            const float u = x[j] - ref, e = __builtin_amdgcn_exp2f(u * kLog2e);
            ls[j & 3] += e;
            ts[j & 3] = fmaf(e, fmaxf(u, -1e30f), ts[j & 3]);
        }
        t = fmaf(r, fmaf(d, l, t), (ts[0] + ts[1]) + (ts[2] + ts[3]));
        l = fmaf(r, l, (ls[0] + ls[1]) + (ls[2] + ls[3]));
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

// The columns of step `step`'s group of lane `tid`: chunk u starts at step * kLpStep + u * 2048 + 8 tid.
__device__ __forceinline__ int64_t lp_column(int64_t group, int u)
{
    return (group / kLpLanes) * kLpStep + u * (kLpLanes * 8) + (group % kLpLanes) * 8;
}

// One lane's part of step `step`: sums into s, returns the group's maximum (NaN if there is one).
template <class IT, bool VEC>
__device__ __forceinline__ float lp_step(const LpArgs& a, const char* base, int64_t step, int tid, LpSum& s)
{
    const int64_t g = step * kLpLanes + tid;
    float x[8 * kLpChunks];
    if (step * kLpStep + kLpStep <= a.n)
    {
        typename IT::Vec v[kLpChunks];
        #pragma unroll
        for (int u = 0; u < kLpChunks; ++u) v[u] = load_chunk<IT, VEC>(base, lp_column(g, u));
        #pragma unroll
        for (int u = 0; u < kLpChunks; ++u)
        {
            float f[8];
            unpack8<IT>(v[u], f);
            #pragma unroll
            for (int j = 0; j < 8; ++j) x[8 * u + j] = f[j];
        }
    }
    else if (a.n >= 8)
    {
        // The row's last columns: a chunk past the end is read so that it ends there, without what belongs to the chunk
        // before (the sums and the maximum ask for no order).
        typename IT::Vec v[kLpChunks];
        #pragma unroll
        for (int u = 0; u < kLpChunks; ++u) v[u] = load_chunk<IT, false>(base, min(lp_column(g, u), a.n - 8));
        #pragma unroll
        for (int u = 0; u < kLpChunks; ++u)
        {
            const int64_t c = lp_column(g, u), at = min(c, a.n - 8);
            float f[8];
            unpack8<IT>(v[u], f);
            #pragma unroll
            for (int j = 0; j < 8; ++j) x[8 * u + j] = at + j >= c ? f[j] : -INFINITY;
        }
    }
    else
    {
        #pragma unroll
        for (int j = 0; j < 8 * kLpChunks; ++j) x[j] = -INFINITY;
        if (g == 0)
        {
            #pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < a.n) x[j] = load1(base, IT::code, j);
        }
    }
    float gm = x[0];
    #pragma unroll
    for (int j = 1; j < 8 * kLpChunks; ++j) gm = lp_max_nan(gm, x[j]);
    float cm = gm;
    if (__any(gm != gm))
    {
        cm = x[0];
        #pragma unroll
        for (int j = 1; j < 8 * kLpChunks; ++j) cm = fmaxf(cm, x[j]);
        cm = cm != cm ? -INFINITY : cm;
    }
    s.add(x, cm);
    return gm;
}

// The workgroup's joined sums, in every lane (lds: 3 floats per wave).
__device__ __forceinline__ LpSum lp_block_sum(LpSum s, float (*w)[3])
{
    #pragma unroll
    for (int d = 1; d < 64; d <<= 1)
    {
        const float m2 = __shfl_xor(s.m, d), l2 = __shfl_xor(s.l, d), t2 = __shfl_xor(s.t, d);
        s.join(m2, l2, t2);
    }
    if ((threadIdx.x & 63) == 0) { w[threadIdx.x >> 6][0] = s.m; w[threadIdx.x >> 6][1] = s.l; w[threadIdx.x >> 6][2] = s.t; }
    __syncthreads();
    s.m = w[0][0]; s.l = w[0][1]; s.t = w[0][2];
    #pragma unroll
    for (int i = 1; i < kLpLanes / 64; ++i) s.join(w[i][0], w[i][1], w[i][2]);
    return s;
}

struct LpShared
{
    u32x4 best[kLpLanes / 4];
    uint32_t list[kLpList];
    uint64_t cand[kLpCands];
    int nlist, nabove, ncand, nfound, count[2];
};

// The order images of a lane's kLpKeep group maxima from group r0 on (0 past the last, below every maximum's): one wait
// for all of them.
template <class P>
__device__ __forceinline__ void lp_maxima(P gmax, int64_t groups, int64_t r0, uint32_t (&k)[kLpKeep])
{
    const int tid = threadIdx.x, left = (int)min(groups - r0, (int64_t)kLpKeep * kLpLanes);
    float v[kLpKeep];
    #pragma unroll
    for (int i = 0; i < kLpKeep; ++i) v[i] = gmax[r0 + min(i * kLpLanes, left - kLpLanes) + tid];     // (left: whole steps)
    #pragma unroll
    for (int i = 0; i < kLpKeep; ++i) k[i] = i * kLpLanes < left ? lp_order(v[i]) : 0;
}

// The row's token and its logit, in one lane of the last wave.
struct LpToken
{
    int64_t id = 0;
    float x = 0.0f;
};
template <class IT>
__device__ __forceinline__ LpToken lp_token(const LpArgs& a, int64_t row)
{
    LpToken t;
    if ((int)threadIdx.x == kLpLanes - 64 && a.tokens)
    {
        t.id = a.tokens[row];
        if (t.id >= 0 && t.id < a.n) t.x = load1(a.x + row * a.ld, IT::code, t.id);
    }
    return t;
}

// Everything a row's sums and group maxima give: m, l, t in every lane; `groups` maxima at gmax, the lane's first ones
// in kept.
template <class IT, class P>
__device__ __forceinline__ void lp_finish(const LpArgs& a, int64_t row, float m, float l, float t, P gmax, int64_t groups,
                                          uint32_t (&kept)[kLpKeep], const LpToken& token, LpShared& sh)
{
    const int tid = threadIdx.x;
    const char* base = a.x + row * a.ld;
    // ln P = (x - m) - ln l: m + ln l would lose ln l beside a large m.  Nothing but -inf: no distribution.
    const double ll = l == 0.0f ? (double)NAN : log((double)l);
    const auto log_p = [&](float x) { return (float)((double)x - m - ll); };
    if (tid == kLpLanes - 64)
    {
        if (a.tokens)
        {
            const int64_t k = token.id;
            if (a.err && (k < 0 || k >= a.vocab)) *a.err = 1;
            a.logprobs[row] = k < 0 || k >= a.n ? (ll != ll ? NAN : -INFINITY) : log_p(token.x);
        }
        if (a.entropy) a.entropy[row] = (float)(ll - (double)t / l);
    }
    const int top = a.top;
    if (!top) return;
    constexpr int64_t ROUND = (int64_t)kLpKeep * kLpLanes;
    uint32_t best = 0;
    for (int64_t r0 = 0; r0 < groups; r0 += ROUND)
    {
        if (r0 != 0) lp_maxima(gmax, groups, r0, kept);
        #pragma unroll
        for (int i = 0; i < kLpKeep; ++i) best = max(best, kept[i]);
    }
    ((uint32_t*)sh.best)[tid] = best;
    if (tid == 0) sh.nlist = sh.nabove = sh.ncand = sh.nfound = 0;
    __syncthreads();
    // The floor: the top-th largest of the lanes' best, as far as its upper 20 bits say (sign, exponent, 11 bits of the
    // fraction): lower by less than 2^-11, a column or two more to rank.  Every wave finds it for itself, bit by bit,
    // four lanes' best in each lane (ranking all against all took 7 of the kernel's 14 us).
    uint32_t floor = 0;
    {
        const u32x4 o = sh.best[tid & 63];
        for (int b = 31; b >= 12; --b)
        {
            const uint32_t w = floor | 1u << b;
            int n = 0;
            #pragma unroll
            for (int j = 0; j < 4; ++j) n += __popcll(__ballot(o[j] >= w));
            floor = n >= top ? w : floor;
        }
    }
    // (a lane without a group that reaches the floor has none to list)
    for (int64_t r0 = 0; r0 < groups && best >= floor; r0 += ROUND)
    {
        if (groups > ROUND) lp_maxima(gmax, groups, r0, kept);
        uint32_t reach = 0, more = 0;
        #pragma unroll
        for (int i = 0; i < kLpKeep; ++i)
        {
            reach |= kept[i] >= floor ? 1u << i : 0u;
            more += kept[i] > floor;
        }
        if (more) atomicAdd(&sh.nabove, more);
        for (int at = reach ? atomicAdd(&sh.nlist, __popc(reach)) : 0; reach; reach &= reach - 1, ++at)
            if (at < kLpList) sh.list[at] = (uint32_t)(r0 + (__ffs(reach) - 1) * kLpLanes + tid);
    }
    __syncthreads();
    const int listed = sh.nlist, above = sh.nabove;
    if (listed <= kLpList)
    {
        constexpr int B = 4;        // (one wait for four of the lane's columns)
        for (int i0 = tid; i0 < listed * kLpChunks * 8; i0 += B * kLpLanes)
        {
            float x[B];
            int64_t c[B];
            #pragma unroll
            for (int u = 0; u < B; ++u)
            {
                const int i = i0 + u * kLpLanes;
                c[u] = i < listed * kLpChunks * 8 ? lp_column(sh.list[i / (kLpChunks * 8)], (i / 8) % kLpChunks) + i % 8 : a.n;
                x[u] = c[u] < a.n ? load1(base, IT::code, c[u]) : 0.0f;
            }
            #pragma unroll
            for (int u = 0; u < B; ++u)
                if (c[u] < a.n && lp_order(x[u]) >= floor)
                {
                    const int at = atomicAdd(&sh.ncand, 1);
                    if (at < kLpCands) sh.cand[at] = lp_key(x[u], (uint32_t)c[u]);
                }
        }
    }
    __syncthreads();
    if (listed > kLpList || sh.ncand > kLpCands)
    {
        // The careful way: many columns share the floor's value (a masked or a constant row), or a few lanes hold many
        // of the largest.  The floor becomes the top-th largest group maximum, unless fewer than top are above it as it is ...
        if (above >= top)
        {
            uint32_t v = 0;
            for (int b = 31; b >= 0; --b)
            {
                const uint32_t w = v | (1u << b);
                int n = 0;
                for (int64_t g = tid; g < groups; g += kLpLanes) n += lp_order(gmax[g]) >= w;
                if (tid == 0) sh.count[b & 1] = 0;
                __syncthreads();
                atomicAdd(&sh.count[b & 1], n);
                __syncthreads();
                if (sh.count[b & 1] >= top) v = w;
            }
            floor = v;
        }
        __syncthreads();
        if (tid == 0) sh.ncand = 0;
        __syncthreads();
        // ... the columns above it are in the fewer than top groups above it ...
        for (int64_t g = tid; g < groups; g += kLpLanes)
            if (lp_order(gmax[g]) > floor)
                for (int u = 0; u < kLpChunks; ++u)
                    for (int64_t c = lp_column(g, u), e = min(c + 8, a.n); c < e; ++c)
                    {
                        const float x = load1(base, IT::code, c);
                        if (lp_order(x) > floor) sh.cand[atomicAdd(&sh.ncand, 1)] = lp_key(x, (uint32_t)c);
                    }
        __syncthreads();
        // ... and the first columns that equal it follow.
        for (int64_t c0 = 0; c0 < a.n; c0 += kLpLanes)
        {
            const int64_t c = c0 + tid;
            const float x = c < a.n ? load1(base, IT::code, c) : 0.0f;
            if (c < a.n && lp_order(x) == floor)
            {
                sh.cand[atomicAdd(&sh.ncand, 1)] = lp_key(x, (uint32_t)c);
                atomicAdd(&sh.nfound, 1);
            }
            __syncthreads();
            const bool done = sh.nfound >= top;
            __syncthreads();
            if (done) break;
        }
    }
    const int n = sh.ncand;
    for (int i = tid; i < n; i += kLpLanes)
    {
        const uint64_t k = sh.cand[i];
        int rank = 0;
        #pragma unroll 8
        for (int j = 0; j < n; ++j) rank += sh.cand[j] > k;
        if (rank < top)
        {
            a.top_ids[row * top + rank] = lp_index(k);
            a.top_logprobs[row * top + rank] = log_p(lp_value(k));
        }
    }
}

// Few rows: a workgroup per slice of a row (a.slices of them, of `steps` steps), sums and maxima to the workspace ...
template <class IT, bool VEC>
__global__ __launch_bounds__(kLpLanes) void k_lp_slices(LpArgs a, int steps)
{
    __shared__ float w[kLpLanes / 64][3];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / (uint32_t)a.slices, sl = blockIdx.x % (uint32_t)a.slices;
    const char* base = a.x + row * a.ld;
    LpSum s;
    for (int64_t i = sl * steps; i < (sl + 1) * steps && i * kLpStep < a.n; ++i)
    {
        const float gm = lp_step<IT, VEC>(a, base, i, tid, s);
        if (a.top) a.gmax[row * a.groups + i * kLpLanes + tid] = gm;
    }
    s = lp_block_sum(s, w);
    if (tid == 0)
    {
        float* p = a.part + 3 * (row * a.slices + sl);
        p[0] = s.m; p[1] = s.l; p[2] = s.t;
    }
}

// ... and a workgroup per row over them.
template <class IT>
__global__ __launch_bounds__(kLpLanes) void k_lp_join(LpArgs a)
{
    __shared__ LpShared sh;
    __shared__ float w[kLpLanes / 64][3];
    const int64_t row = blockIdx.x;
    const gcptr<float> gmax = (gcptr<float>)a.gmax + row * a.groups;
    const LpToken token = lp_token<IT>(a, row);
    uint32_t kept[kLpKeep] = {};
    if (a.top) lp_maxima(gmax, a.groups, 0, kept);
    LpSum s;
    if ((int)threadIdx.x < a.slices)
    {
        const gcptr<float> p = (gcptr<float>)a.part + 3 * (row * a.slices + threadIdx.x);
        s.m = p[0]; s.l = p[1]; s.t = p[2];
    }
    s = lp_block_sum(s, w);
    lp_finish<IT>(a, row, s.m, s.l, s.t, gmax, a.groups, kept, token, sh);
}

// Many rows: a workgroup per row, its group maxima in LDS.
template <class IT, bool VEC>
__global__ __launch_bounds__(kLpLanes) void k_lp_rows(LpArgs a)
{
    extern __shared__ float gmax[];
    __shared__ LpShared sh;
    __shared__ float w[kLpLanes / 64][3];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const char* base = a.x + row * a.ld;
    const LpToken token = lp_token<IT>(a, row);
    LpSum s;
    for (int64_t i = 0; i * kLpStep < a.n; ++i)
    {
        const float gm = lp_step<IT, VEC>(a, base, i, tid, s);
        if (a.top) gmax[i * kLpLanes + tid] = gm;
    }
    s = lp_block_sum(s, w);
    uint32_t kept[kLpKeep] = {};
    if (a.top) lp_maxima(gmax, a.groups, 0, kept);
    lp_finish<IT>(a, row, s.m, s.l, s.t, gmax, a.groups, kept, token, sh);
}

}  // namespace exl3r

using namespace exl3r;

namespace {

struct LpPlan
{
    bool by_rows;
    int64_t steps, slices, groups;      // steps per slice
    size_t part_bytes, bytes;
};

LpPlan lp_plan(int64_t rows, int64_t n)
{
    LpPlan p;
    const int64_t all = (n + kLpStep - 1) / kLpStep;
    p.groups = all * kLpLanes;
    // A workgroup per row from one row per CU on (slices / rows: 32003 f16 columns, 192 rows 9.8 / 9.5 us, 128 rows 8.2 /
    // 9.5; 151936 fp32 columns with 20 alternatives, 256 rows 38 / 36 us, 192 rows 31 / 35), if the group maxima leave
    // room for two in the LDS.
    p.by_rows = rows >= 256 && p.groups * 4 <= 64 << 10;
    p.steps = (all + 255) / 256;
    p.slices = (all + p.steps - 1) / p.steps;
    // (as if for the most slices: fewer columns then never ask for more)
    p.part_bytes = ((size_t)rows * (all < 256 ? all : 256) * 12 + 255) & ~(size_t)255;
    p.bytes = p.by_rows ? 0 : p.part_bytes + (size_t)rows * p.groups * 4;
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
    if (p.bytes && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < p.bytes))
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
    const bool vec = aligned16(logits) && a.ld % 16 == 0;
    if (!p.by_rows && rows * p.slices > 0xffffff) return set_error(EXL3R_EINVAL, "%s: more than 2^24 workgroups", op);
    with_float_type(dtype, [&](auto T) {
        using Ty = decltype(T);
        if (p.by_rows)
        {
            const size_t lds = top_k ? (size_t)p.groups * 4 : 0;
            if (vec) launch(k_lp_rows<Ty, true>, (unsigned)rows, kLpLanes, lds, s, a);
            else launch(k_lp_rows<Ty, false>, (unsigned)rows, kLpLanes, lds, s, a);
            return;
        }
        if (vec) launch(k_lp_slices<Ty, true>, (unsigned)(rows * p.slices), kLpLanes, 0, s, a, (int)p.steps);
        else launch(k_lp_slices<Ty, false>, (unsigned)(rows * p.slices), kLpLanes, 0, s, a, (int)p.steps);
        launch(k_lp_join<Ty>, (unsigned)rows, kLpLanes, 0, s, a);
    });
    return launch_status(op);
}
