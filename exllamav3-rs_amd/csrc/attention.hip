// Attention over the paged KV cache for gfx950: exl3r_paged_attn and exl3r_paged_attn_shared.
//
// Token s of sequence b is at position p = cache_seqlens[b] + s (the place where exl3r_rope_paged_kv put it);
// it sees the keys j <= p that are inside the window (p - j < window) or among the first `sinks` positions.
//   S = q . k_j;  o = sum_j 2^(c S_j - c m) v_j / sum_j 2^(c S_j - c m),  c = scale log2 e, m the row's maximum,
// in one pass over the keys with the running m, l (the sum) and o of each query row in fp32 registers.
//
// Both products run on the matrix cores as v_mfma_f32_32x32x16 with the query rows as columns:
//   S^T[key, row] = K Q^T,   o^T[d, row] = V^T P^T.
// A lane then holds 16 of a 32-key tile's scores of ONE query row (lane l: row l % 32, keys 8 (i / 4) + 4 (l / 32)
// + i % 4), so the softmax needs no cross-lane step but one swap with lane l ^ 32, and the packed probabilities
// are already the second product's B operand if V^T's keys are taken in the same order, which is what the
// transposing LDS read (ds_read_b64_tr_b16) delivers: 4 consecutive keys of one column per read.
// A query row of the kernels is a (token, query head) pair: the heads that share a KV head are packed together,
// so one read of K and V serves the whole group.
#include "abi.hpp"
#include "common.cuh"

namespace exl3r {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <class T> using lptr = __attribute__((address_space(3))) T*;

constexpr int kMaxSplits = 512;      // of a row: 256 of the shared prefix and 256 of its own keys

struct AttnArgs
{
    const char* q;
    char* out;
    float* lse;               // nullptr: not written
    const char* kc;
    const char* vc;
    const int32_t* table;
    const int32_t* lens;
    int32_t* err;
    float* po;                // partial outputs [row][split][HD], unnormalised
    float* pml;               // ... and their {c m - shift, l} [row][split][2]
    int64_t q_ts, q_hs, o_ts, o_hs;     // elements
    int64_t max_blocks, num_pages;
    int64_t rows_all;         // bsz * seq * hq
    int32_t bsz, seq, hq, hk, group;
    int32_t page_shift, window, sinks;
    int32_t dom_lo, dom_hi;   // keys of this launch: [dom_lo, dom_hi)
    int32_t rows;             // query rows per row set (a sequence's, or the whole batch's)
    int32_t row_tiles, nsplit, split0, splits;   // this launch's splits, their first place among all `splits`
    int32_t whole;            // 1: one row set of all sequences, keys through sequence 0's table row
    int32_t direct;           // 1: this launch's result is the output
    int32_t q_vec, o_vec;     // 16-byte aligned q rows / 8-byte aligned out rows
    float c;
};

template <class IO>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (IO::code == DT_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <class IO>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (IO::code == DT_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <class IO>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    if constexpr (IO::code == DT_F16) return pack_f16(lo, hi);
    else return pack_bf16(lo, hi);
}

// v(l) and v(l ^ 32) combined, the same in both lanes.
__device__ __forceinline__ float max_xor32(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1]));
}

// ... of the four lanes l % 16 + {0, 16, 32, 48}.
__device__ __forceinline__ float max_xor16(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1]));
}

// Orders LDS accesses of one wave's lanes (no instruction: a wave's LDS accesses execute in order).
__device__ __forceinline__ void wave_lds_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// LDS layout of a tile of K or V: rows of HD elements, the 16-byte chunks of row `key` permuted by an XOR with
// swz(key), which puts the 16 rows that a K read touches (one chunk column) and the 4 x 64 bytes of a
// transposing V read on different banks.
template <int HD>
__device__ __forceinline__ int swz(int key)
{
    if constexpr (HD == 64) return (((key >> 1) & 1) << 2) | ((key >> 2) & 3);
    else return ((key & 3) << 2) | ((key >> 2) & 3);
}

// A query row: its token and head, its position.
struct QRow
{
    int64_t tok;
    int h, p;
};

__device__ __forceinline__ QRow query_row(const AttnArgs& a, int set, int kvh, int r)
{
    const int t = r / a.group;
    QRow q;
    q.h = kvh * a.group + (r - t * a.group);
    const int b = a.whole ? t / a.seq : set;
    const int s = a.whole ? t - b * a.seq : t;
    q.tok = (int64_t)b * a.seq + s;
    const int64_t p = (int64_t)a.lens[b] + s;
    q.p = p > 0x7fffffff ? 0x7fffffff : p < -1 ? -1 : (int)p;
    return q;
}

__device__ __forceinline__ int wave_min(int v)
{
    #pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = min(v, __shfl_xor(v, d));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max(int v)
{
    #pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = max(v, __shfl_xor(v, d));
    return __builtin_amdgcn_readfirstlane(v);
}

__device__ __forceinline__ float max_wave(float v)
{
    #pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

// The key tiles (KT keys from dom_lo on) that some row with a position in [pmin, pmax] sees: `ns` tiles of
// sinks, then the tiles from wt on; and the part [it0, it1) of that list that a split takes.
struct TileList
{
    int ns, wt, count, khi;
    __device__ __forceinline__ int tile(int it) const { return it < ns ? it : wt + (it - ns); }
};

__device__ __forceinline__ TileList tile_list(const AttnArgs& a, int pmin, int pmax, int kt)
{
    TileList l;
    l.khi = min(a.dom_hi, pmax < 0x7fffffff ? pmax + 1 : pmax);
    const int n = l.khi - a.dom_lo;
    if (n <= 0) { l.ns = l.wt = l.count = 0; return l; }
    const int ht = (n + kt - 1) / kt;
    const int64_t lo = a.window > 0 ? (int64_t)pmin - a.window + 1 - a.dom_lo : 0;
    l.wt = lo > 0 ? min((int)lo / kt, ht) : 0;
    l.ns = a.window > 0 ? min(l.wt, max(0, (min(a.sinks, l.khi) - a.dom_lo + kt - 1) / kt)) : 0;
    l.count = l.ns + ht - l.wt;
    return l;
}

// Whether some row from position pmin on sees key j: the page table is trusted for no other (pages behind every
// window may be gone).
__device__ __forceinline__ bool key_seen(const AttnArgs& a, const TileList& l, int j, int pmin)
{
    return j < l.khi && (a.window <= 0 || pmin - j < a.window || j < a.sinks);
}

// State of 32 query rows (a lane's row, its half of the scores and of o's rows).
template <int HD>
struct Acc
{
    f32x16 o[HD / 32];
    float m, l;
    __device__ __forceinline__ void clear()
    {
        #pragma unroll
        for (int t = 0; t < HD / 32; ++t)
            #pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
        m = -INFINITY;
        l = 0.0f;
    }
};

// A row's B operand for steps of DK dimensions: part `part` of each step's 8-element parts.
template <class IO, int HD, int DK>
__device__ __forceinline__ void load_q(const AttnArgs& a, const QRow& r, int part, u32x4 (&qf)[HD / DK])
{
    const uint16_t* src = (const uint16_t*)a.q + r.tok * a.q_ts + (int64_t)r.h * a.q_hs;
    #pragma unroll
    for (int t = 0; t < HD / DK; ++t)
    {
        const int e = DK * t + 8 * part;
        if (a.q_vec) qf[t] = *(gcptr<u32x4>)(src + e);
        else
        {
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                qf[t][i] = (uint32_t)((gcptr<uint16_t>)src)[e + 2 * i] | (uint32_t)((gcptr<uint16_t>)src)[e + 2 * i + 1] << 16;
        }
    }
}

// Four elements of an output row.
template <class IO>
__device__ __forceinline__ void store_out4(const AttnArgs& a, int64_t tok, int h, int d, float x, float y, float z, float w)
{
    const gptr<uint16_t> p = (gptr<uint16_t>)((uint16_t*)a.out + tok * a.o_ts + (int64_t)h * a.o_hs + d);
    const u32x2 v = { pack2<IO>(x, y), pack2<IO>(z, w) };
    if (a.o_vec) *(gptr<u32x2>)p = v;
    else
    {
        p[0] = (uint16_t)v.x; p[1] = (uint16_t)(v.x >> 16);
        p[2] = (uint16_t)v.y; p[3] = (uint16_t)(v.y >> 16);
    }
}

// S^T of 32 keys (LDS rows from kb on) and the lane's 32-row column tile.
template <class IO, int HD>
__device__ __forceinline__ f32x16 qk_tile(const char* kb, int lane, const u32x4 (&qf)[HD / 16])
{
    const int key = lane & 31, half = lane >> 5;
    const char* row = kb + key * (HD * 2);
    const int x = (swz<HD>(key) ^ half) << 4;
    f32x16 s{};
    #pragma unroll
    for (int t = 0; t < HD / 16; ++t)
    {
        const u32x4 kf = *(const u32x4*)(row + (x ^ (t << 5)));
        s = mfma32<IO>(kf, qf[t], s);
    }
    return s;
}

// Which of the 32 keys from j0 on the lane's row sees: its scores elsewhere become -inf.
__device__ __forceinline__ void mask_tile(f32x16& s, int j0, int half, int p, int window, int sinks, uint32_t ok)
{
    const int lo = window > 0 ? p - window + 1 : 0;
    const int jb = j0 + 4 * half;
    const uint32_t okh = ok >> (4 * half);
    #pragma unroll
    for (int i = 0; i < 16; ++i)
    {
        const int d = 8 * (i / 4) + i % 4, j = jb + d;
        const bool see = (j <= p) & ((j >= lo) | (j < sinks)) & (((okh >> d) & 1u) != 0);
        s[i] = see ? s[i] : -INFINITY;
    }
}

// Exponents of the probabilities are raised by kShift: as f16, whose smallest normal number is 2^-14, a probability
// keeps its 11 bits down to 2^-28 of the row's largest (bf16 has fp32's range).  o and l carry the same factor.
template <class IO> constexpr float kShift = IO::code == DT_F16 ? 14.0f : 0.0f;

// The running softmax over one more tile of scores: s becomes the probabilities against the new maximum.
template <class IO, int HD>
__device__ __forceinline__ void softmax_tile(Acc<HD>& a, f32x16& s, float c)
{
    float mx = s[0];
    #pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    const float mn = fmaxf(a.m, max_xor32(mx));
    const float ref = (mn == -INFINITY ? 0.0f : mn) * c;
    const float alpha = __builtin_amdgcn_exp2f(fmaf(a.m, c, -ref));
    float sum = 0.0f;
    #pragma unroll
    for (int i = 0; i < 16; ++i)
    {
        s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, kShift<IO> - ref));
        sum += s[i];
    }
    a.l = fmaf(a.l, alpha, sum);
    a.m = mn;
    #pragma unroll
    for (int t = 0; t < HD / 32; ++t)
        #pragma unroll
        for (int i = 0; i < 16; ++i) a.o[t][i] *= alpha;
}

// Whether some of 8 elements of V is an infinity or a NaN.
template <class IO>
__device__ __forceinline__ bool nonfinite8(const u32x4& v)
{
    constexpr uint32_t E = IO::code == DT_F16 ? 0x7c00u : 0x7f80u, E2 = E | E << 16, B = E & (0u - E), B2 = B | B << 16;
    uint32_t c = 0;     // the carry of exponent + 1 out of the exponent's field: all ones there
    #pragma unroll
    for (int i = 0; i < 4; ++i) c |= ((v[i] & E2) + B2) & 0x80008000u;
    return c != 0;
}

// Zeroes the infinities and NaNs of v and returns their indicators: 1 for +inf, 64 for -inf, 65 for a NaN.
template <class IO>
__device__ __forceinline__ u32x4 take_nonfinite(u32x4& v)
{
    constexpr uint32_t E = IO::code == DT_F16 ? 0x7c00u : 0x7f80u;
    u32x4 ind;
    #pragma unroll
    for (int e = 0; e < 4; ++e)
    {
        float w[2];
        uint32_t keep = 0;
        #pragma unroll
        for (int k = 0; k < 2; ++k)
        {
            const uint32_t h = ((uint32_t)v[e] >> (16 * k)) & 0xffffu, mag = h & 0x7fffu;
            w[k] = mag > E ? 65.0f : mag < E ? 0.0f : h >> 15 ? 64.0f : 1.0f;
            keep |= mag < E ? 0xffffu << (16 * k) : 0u;
        }
        ind[e] = pack2<IO>(w[0], w[1]);
        v[e] &= keep;
    }
    return ind;
}
// What n = (count of +inf) + 64 (count of -inf), NaNs in both, adds to a sum.
__device__ __forceinline__ float nonfinite_sum(float n)
{
    const int c = (int)n;
    return (c & 63 ? INFINITY : 0.0f) - (c >> 6 ? INFINITY : 0.0f);
}

// o^T += V^T P^T over 32 keys (LDS rows from vb on).  The probabilities are rounded to V's type for the matrix
// cores: one rounding of at most half a step each, against the same maximum for the whole row; l sums them
// unrounded.  CARE: V has infinities or NaNs and some row does not see some of these keys; there the probability
// is 0, but 0 * inf and 0 * NaN must not reach the row.  They are then taken out of the product and applied by a
// second one, of 1 where V has +inf or NaN, 64 where it has -inf or NaN and 65 for a NaN, with "the row's probability
// is not 0": its sums over at most 32 keys tell how many of each a row sees.
template <class IO, int HD, bool CARE>
__device__ __forceinline__ void pv_tile(Acc<HD>& a, const f32x16& p, const char* vb, int lane)
{
    const int i16 = lane & 15, half = lane >> 5;
    const int key = 4 * half + (i16 >> 2);
    const int c0 = ((lane >> 3) & 2) | ((i16 >> 1) & 1);
    const char* r0 = vb + key * (HD * 2) + ((i16 & 1) << 3);
    const int x0 = (swz<HD>(key) ^ c0) << 4, x1 = (swz<HD>(key + 8) ^ c0) << 4;
    #pragma unroll
    for (int u = 0; u < 2; ++u)
    {
        u32x4 pf, see{};
        #pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            pf[e] = pack2<IO>(p[8 * u + 2 * e], p[8 * u + 2 * e + 1]);
            if constexpr (CARE)
                see[e] = pack2<IO>(p[8 * u + 2 * e] != 0.0f ? 1.0f : 0.0f, p[8 * u + 2 * e + 1] != 0.0f ? 1.0f : 0.0f);
        }
        #pragma unroll
        for (int t = 0; t < HD / 32; ++t)
        {
            const auto v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr<s16x4>)(r0 + u * 16 * HD * 2 + (x0 ^ (t << 6))));
            const auto v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr<s16x4>)(r0 + (u * 16 + 8) * HD * 2 + (x1 ^ (t << 6))));
            const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
            u32x4 vf = { w0.x, w0.y, w1.x, w1.y };
            if constexpr (CARE)
            {
                const u32x4 ind = take_nonfinite<IO>(vf);
                f32x16 n{};
                n = mfma32<IO>(ind, see, n);
                #pragma unroll
                for (int i = 0; i < 16; ++i) a.o[t][i] += nonfinite_sum(n[i]);
            }
            a.o[t] = mfma32<IO>(vf, pf, a.o[t]);
        }
    }
}

// The page of key j (-1 past the keys of the launch).
__device__ __forceinline__ int page_entry(const AttnArgs& a, const int32_t* table, int j, int khi)
{
    return j < khi ? table[j >> a.page_shift] : -1;
}

// One tile's loads.  SMALL (pages of fewer keys than a tile): a lane's key has a page of its own, entry k of the
// tile's page list being in lane k.  Otherwise the tile lies in one page, at a wave-uniform base, and the keys past
// the last one are read too (they are in the page) and taken out later.  A bad page's keys read page 0.
template <int HD, bool SMALL, int STEPS, int LANES>
__device__ __forceinline__ void load_tile(const AttnArgs& a, int j0, int entry, uint64_t ok, int kvh, int lane_of_tile,
                                          u32x4 (&ks)[STEPS], u32x4 (&vs)[STEPS])
{
    constexpr int CH = HD / 8, KPS = LANES / CH;      // keys per step
    const int key0 = lane_of_tile / CH, ch = lane_of_tile % CH;
    const uint32_t row_bytes = (uint32_t)a.hk * (HD * 2);
    const int in_page = (1 << a.page_shift) - 1;
    if constexpr (SMALL)
    {
        #pragma unroll
        for (int k = 0; k < STEPS; ++k)
        {
            const int key = k * KPS + key0, page = __shfl(entry, key);
            const int64_t row = (ok >> key) & 1 ? ((int64_t)page << a.page_shift) + ((j0 + key) & in_page) : 0;
            const int64_t off = row * row_bytes + kvh * (HD * 2) + ch * 16;
            ks[k] = *(gcptr<u32x4>)(a.kc + off);
            vs[k] = *(gcptr<u32x4>)(a.vc + off);
        }
    }
    else
    {
        const int page = __builtin_amdgcn_readfirstlane(entry);
        const int64_t row = (ok ? (int64_t)page << a.page_shift : 0) + (j0 & in_page);
        const int64_t base = row * row_bytes + kvh * (HD * 2);
        const uint32_t off = key0 * row_bytes + ch * 16;
        #pragma unroll
        for (int k = 0; k < STEPS; ++k)
        {
            const int64_t b = base + (int64_t)(k * KPS) * row_bytes;
            ks[k] = *(gcptr<u32x4>)(a.kc + b + off);
            vs[k] = *(gcptr<u32x4>)(a.vc + b + off);
        }
    }
}

// The launch's item: KV head (fastest: consecutive workgroups go to different XCDs, so with 8 KV heads an XCD's
// L2 holds the keys of one head), then row tile (the last, longest first), split, row set.
struct Item
{
    int kvh, tile, split, set;
};
__device__ __forceinline__ Item launch_item(const AttnArgs& a)
{
    uint32_t x = blockIdx.x;
    Item it;
    it.kvh = x % (uint32_t)a.hk;
    x /= (uint32_t)a.hk;
    it.tile = a.row_tiles - 1 - (int)(x % (uint32_t)a.row_tiles);
    x /= (uint32_t)a.row_tiles;
    it.split = x % (uint32_t)a.nsplit;
    it.set = x / (uint32_t)a.nsplit;
    return it;
}

__device__ __forceinline__ void flag_positions(const AttnArgs& a, const QRow& r)
{
    const int64_t cap = a.max_blocks << a.page_shift;
    if (a.err && (r.p < 0 || r.p >= cap)) *a.err = 1;
}

// ---------------------------------------------------------------------------------------------
// Many query rows: 4 waves of NQ * 32 rows each share tiles of 64 keys in LDS; the next tile's loads are in
// flight (registers) while a tile is multiplied.
template <class IO, int HD, int NQ, bool SMALL>
__global__ __launch_bounds__(256, HD == 256 || NQ == 2 ? 1 : 2) void k_attn_rows(AttnArgs a)
{
    constexpr int KT = 64, CH = HD / 8, RB = HD * 2, STEPS = KT * CH / 256;
    __shared__ __align__(16) char lds[2 * KT * RB];
    char* const kl = lds;
    char* const vl = lds + KT * RB;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const Item it = launch_item(a);

    QRow row[NQ];
    u32x4 qf[NQ][HD / 16];
    Acc<HD> acc[NQ];
    int pmin[NQ], pmax[NQ];
    const int r0 = it.tile * (128 * NQ) + wave * (32 * NQ);
    #pragma unroll
    for (int n = 0; n < NQ; ++n)
    {
        row[n] = query_row(a, it.set, it.kvh, min(r0 + 32 * n + (lane & 31), a.rows - 1));
        load_q<IO, HD, 16>(a, row[n], half, qf[n]);
        acc[n].clear();
        pmin[n] = wave_min(row[n].p);
        pmax[n] = wave_max(row[n].p);
        if (it.split == 0 && it.kvh == 0) flag_positions(a, row[n]);
    }
    // positions of the whole workgroup's rows
    __shared__ int plo[4], phi[4], odd[2];
    int wmin = pmin[0], wmax = pmax[0];
    #pragma unroll
    for (int n = 1; n < NQ; ++n) { wmin = min(wmin, pmin[n]); wmax = max(wmax, pmax[n]); }
    if (lane == 0) { plo[wave] = wmin; phi[wave] = wmax; }
    if (tid == 0) odd[0] = odd[1] = 0;
    __syncthreads();
    const int gmin = min(min(plo[0], plo[1]), min(plo[2], plo[3]));
    const int gmax = max(max(phi[0], phi[1]), max(phi[2], phi[3]));
    const TileList tl = tile_list(a, gmin, gmax, KT);
    const int per = (tl.count + a.nsplit - 1) / a.nsplit;
    const int t0 = min(it.split * per, tl.count), t1 = min(t0 + per, tl.count);

    const int32_t* table = a.table + (a.whole ? 0 : (int64_t)it.set * a.max_blocks);
    u32x4 ks[STEPS], vs[STEPS];
    int entry = -1;
    uint64_t ok_next = 0;
    auto fetch_entry = [&](int i) { entry = i < t1 ? page_entry(a, table, a.dom_lo + tl.tile(i) * KT + lane, tl.khi) : -1; };
    auto stage = [&](int i) {
        const int j0 = a.dom_lo + tl.tile(i) * KT;
        const bool in = key_seen(a, tl, j0 + lane, gmin), good = in && (uint64_t)(int64_t)entry < (uint64_t)a.num_pages;
        if (a.err && in && !good) *a.err = 1;
        ok_next = __ballot(good);
        load_tile<HD, SMALL, STEPS, 256>(a, j0, entry, ok_next, it.kvh, tid, ks, vs);
    };
    fetch_entry(t0);
    if (t0 < t1) { stage(t0); fetch_entry(t0 + 1); }
    for (int i = t0; i < t1; ++i)
    {
        const uint64_t ok = ok_next;
        const int j0 = a.dom_lo + tl.tile(i) * KT;
        const bool all = ok == ~0ull && j0 + KT - 1 <= gmin && (a.window <= 0 || gmax - j0 < a.window || j0 + KT - 1 < a.sinks);
        __syncthreads();
        bool nf = false;
        if (!all)
        {
            #pragma unroll
            for (int k = 0; k < STEPS; ++k)
            {
                if (!((ok >> ((k * 256 + tid) / CH)) & 1)) ks[k] = vs[k] = u32x4{};
                nf |= nonfinite8<IO>(vs[k]);
            }
        }
        #pragma unroll
        for (int k = 0; k < STEPS; ++k)
        {
            const int slot = k * 256 + tid, key = slot / CH, ch = slot % CH;
            const int at = key * RB + ((ch ^ swz<HD>(key)) << 4);
            *(u32x4*)(kl + at) = ks[k];
            *(u32x4*)(vl + at) = vs[k];
        }
        // odd[i & 1]: V of this tile has infinities or NaNs and not every row sees all of it
        if (nf) odd[i & 1] = 1;
        if (tid == 0) odd[(i + 1) & 1] = 0;
        __syncthreads();
        const bool care = odd[i & 1] != 0;
        if (i + 1 < t1) { stage(i + 1); fetch_entry(i + 2); }
        #pragma unroll
        for (int n = 0; n < NQ; ++n)
        {
            #pragma unroll
            for (int k = 0; k < 2; ++k)
            {
                const int j = j0 + 32 * k;
                const uint32_t okw = (uint32_t)(ok >> (32 * k));
                const bool none = okw == 0 || j > pmax[n] || (a.window > 0 && pmin[n] - (j + 31) >= a.window && j >= a.sinks);
                if (none) continue;
                const bool whole = okw == 0xffffffffu && j + 31 <= pmin[n] &&
                                   (a.window <= 0 || pmax[n] - j < a.window || j + 31 < a.sinks);
                f32x16 s = qk_tile<IO, HD>(kl + k * 32 * RB, lane, qf[n]);
                if (!whole) mask_tile(s, j, half, row[n].p, a.window, a.sinks, okw);
                softmax_tile<IO, HD>(acc[n], s, a.c);
                if (!care) pv_tile<IO, HD, false>(acc[n], s, vl + k * 32 * RB, lane);
                else pv_tile<IO, HD, true>(acc[n], s, vl + k * 32 * RB, lane);
            }
        }
    }
    #pragma unroll
    for (int n = 0; n < NQ; ++n)
    {
        const int r = r0 + 32 * n + (lane & 31);
        const float l = sum_xor32(acc[n].l);
        if (r >= a.rows) continue;
        const int64_t gr = row[n].tok * a.hq + row[n].h;
        if (a.direct)
        {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            if (a.lse && half == 0) a.lse[gr] = l == 0.0f ? -INFINITY : (fmaf(acc[n].m, a.c, -kShift<IO>) + __builtin_amdgcn_logf(l)) * 0.69314718055994530942f;
            #pragma unroll
            for (int t = 0; t < HD / 32; ++t)
                #pragma unroll
                for (int g = 0; g < 4; ++g)
                    store_out4<IO>(a, row[n].tok, row[n].h, 32 * t + 8 * g + 4 * half, acc[n].o[t][4 * g] * inv,
                                   acc[n].o[t][4 * g + 1] * inv, acc[n].o[t][4 * g + 2] * inv, acc[n].o[t][4 * g + 3] * inv);
        }
        else
        {
            const int64_t pr = gr * a.splits + a.split0 + it.split;
            if (half == 0) { a.pml[2 * pr] = fmaf(acc[n].m, a.c, -kShift<IO>); a.pml[2 * pr + 1] = l; }
            if (l == 0.0f) continue;
            gptr<f32x4> d = (gptr<f32x4>)(a.po + pr * HD + 4 * half);
            #pragma unroll
            for (int t = 0; t < HD / 32; ++t)
                #pragma unroll
                for (int g = 0; g < 4; ++g)
                    d[8 * t + 2 * g] = f32x4{ acc[n].o[t][4 * g], acc[n].o[t][4 * g + 1], acc[n].o[t][4 * g + 2], acc[n].o[t][4 * g + 3] };
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Few query rows (decode): the 4 waves of a workgroup hold the same NC * 16 rows and walk different tiles of 32 keys,
// each through its own part of LDS without a barrier; their results are joined at the end.  With 16 rows per MFMA
// column tile (v_mfma_f32_16x16x32: lane l holds row l % 16, keys 4 (l / 16) + i of each 16) a group of 8 or 16 query
// heads leaves little of a tile empty, and o, Q and the scores take half the registers of 32 rows, so that two tiles
// of loads per SIMD stay in flight: HBM is the bound here.
template <class IO, int HD, int NC, bool SMALL>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void k_attn_keys(AttnArgs a)
{
    constexpr int KT = 32, CH = HD / 8, RB = HD * 2, STEPS = KT * CH / 64, ROWS = 16 * NC;
    __shared__ __align__(16) char lds[4][2 * KT * RB];
    __shared__ float mlw[4][2][ROWS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4, col = lane & 15;
    char* const kl = lds[wave];
    char* const vl = lds[wave] + KT * RB;
    const Item it = launch_item(a);
    const int r0 = it.tile * ROWS;
    QRow row[NC];
    int pmin = 0x7fffffff, pmax = -0x7fffffff;
    #pragma unroll
    for (int n = 0; n < NC; ++n)
    {
        row[n] = query_row(a, it.set, it.kvh, min(r0 + 16 * n + col, a.rows - 1));
        if (it.split == 0 && it.kvh == 0) flag_positions(a, row[n]);
        pmin = min(pmin, row[n].p);
        pmax = max(pmax, row[n].p);
    }
    pmin = wave_min(pmin);
    pmax = wave_max(pmax);
    const TileList tl = tile_list(a, pmin, pmax, KT);
    const int per = ((tl.count + a.nsplit - 1) / a.nsplit + 3) & ~3;
    const int t0 = min(it.split * per, tl.count), t1 = min(t0 + per, tl.count);

    const int32_t* table = a.table + (a.whole ? 0 : (int64_t)it.set * a.max_blocks);
    u32x4 ks[STEPS], vs[STEPS];
    int entry = -1;
    uint32_t ok_next = 0;
    auto fetch_entry = [&](int i) {
        entry = i < t1 ? page_entry(a, table, a.dom_lo + tl.tile(i) * KT + (lane & 31), tl.khi) : -1;
    };
    auto stage = [&](int i) {
        const int j0 = a.dom_lo + tl.tile(i) * KT;
        const bool in = key_seen(a, tl, j0 + (lane & 31), pmin), good = in && (uint64_t)(int64_t)entry < (uint64_t)a.num_pages;
        if (a.err && in && !good) *a.err = 1;
        ok_next = (uint32_t)__ballot(good);
        load_tile<HD, SMALL, STEPS, 64>(a, j0, entry, ok_next, it.kvh, lane, ks, vs);
    };
    fetch_entry(t0 + wave);
    if (t0 + wave < t1) { stage(t0 + wave); fetch_entry(t0 + wave + 4); }

    u32x4 qf[NC][HD / 32];
    f32x4 o[NC][HD / 16];
    float m[NC], l[NC];
    #pragma unroll
    for (int n = 0; n < NC; ++n)
    {
        load_q<IO, HD, 32>(a, row[n], quad, qf[n]);
        #pragma unroll
        for (int t = 0; t < HD / 16; ++t) o[n][t] = f32x4{};
        m[n] = -INFINITY;
        l[n] = 0.0f;
    }
    // K fragment: key row col (of 16), chunks 4 t + quad; V^T fragment: keys 4 quad + 0..3 (and + 16), columns 16 t + col
    const char* const krow = kl + col * RB;
    const int kx = (swz<HD>(col) ^ quad) << 4;
    const int vkey = 4 * quad + (col >> 2);
    const char* const vrow = vl + vkey * RB + ((col & 1) << 3);
    const int vx = (swz<HD>(vkey) ^ ((col >> 1) & 1)) << 4;
    for (int i = t0 + wave; i < t1; i += 4)
    {
        const uint32_t ok = ok_next;
        const int j = a.dom_lo + tl.tile(i) * KT;
        const bool whole = ok == 0xffffffffu && j + 31 <= pmin && (a.window <= 0 || pmax - j < a.window || j + 31 < a.sinks);
        bool nf = false;
        wave_lds_fence();
        if (!whole)
        {
            #pragma unroll
            for (int k = 0; k < STEPS; ++k)
            {
                if (!((ok >> ((k * 64 + lane) / CH)) & 1)) ks[k] = vs[k] = u32x4{};
                nf |= nonfinite8<IO>(vs[k]);
            }
        }
        #pragma unroll
        for (int k = 0; k < STEPS; ++k)
        {
            const int slot = k * 64 + lane, key = slot / CH, ch = slot % CH;
            const int at = key * RB + ((ch ^ swz<HD>(key)) << 4);
            *(u32x4*)(kl + at) = ks[k];
            *(u32x4*)(vl + at) = vs[k];
        }
        const bool care = __any(nf);
        wave_lds_fence();
        if (i + 4 < t1) { stage(i + 4); fetch_entry(i + 8); }
        if (ok == 0) continue;
        f32x4 s[NC][2];
        #pragma unroll
        for (int k = 0; k < 2; ++k)
        {
            #pragma unroll
            for (int n = 0; n < NC; ++n) s[n][k] = f32x4{};
            #pragma unroll
            for (int t = 0; t < HD / 32; ++t)
            {
                const u32x4 kf = *(const u32x4*)(krow + k * 16 * RB + (kx ^ (t << 6)));
                #pragma unroll
                for (int n = 0; n < NC; ++n) s[n][k] = mfma16<IO>(kf, qf[n][t], s[n][k]);
            }
        }
        u32x4 pf[NC], see[NC];
        #pragma unroll
        for (int n = 0; n < NC; ++n)
        {
            if (!whole)
            {
                const int p = row[n].p, lo = a.window > 0 ? p - a.window + 1 : 0;
                const uint32_t okq = ok >> (4 * quad);
                #pragma unroll
                for (int k = 0; k < 2; ++k)
                    #pragma unroll
                    for (int e = 0; e < 4; ++e)
                    {
                        const int jj = j + 4 * quad + 16 * k + e;
                        const bool vis = (jj <= p) & ((jj >= lo) | (jj < a.sinks)) & (((okq >> (16 * k + e)) & 1u) != 0);
                        s[n][k][e] = vis ? s[n][k][e] : -INFINITY;
                    }
            }
            float mx = s[n][0][0];
            #pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[n][e >> 2][e & 3]);
            const float mn = fmaxf(m[n], max_xor32(max_xor16(mx)));
            const float ref = (mn == -INFINITY ? 0.0f : mn) * a.c;
            const float alpha = __builtin_amdgcn_exp2f(fmaf(m[n], a.c, -ref));
            float sum = 0.0f, pr[8];
            #pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                pr[e] = __builtin_amdgcn_exp2f(fmaf(s[n][e >> 2][e & 3], a.c, kShift<IO> - ref));
                sum += pr[e];
            }
            l[n] = fmaf(l[n], alpha, sum);
            m[n] = mn;
            #pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                pf[n][e] = pack2<IO>(pr[2 * e], pr[2 * e + 1]);
                see[n][e] = pack2<IO>(pr[2 * e] != 0.0f ? 1.0f : 0.0f, pr[2 * e + 1] != 0.0f ? 1.0f : 0.0f);
            }
            #pragma unroll
            for (int t = 0; t < HD / 16; ++t)
                #pragma unroll
                for (int e = 0; e < 4; ++e) o[n][t][e] *= alpha;
        }
        #pragma unroll
        for (int t = 0; t < HD / 16; ++t)
        {
            const auto v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr<s16x4>)(vrow + (vx ^ (t << 5))));
            const auto v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr<s16x4>)(vrow + 16 * RB + (vx ^ (t << 5))));
            const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
            u32x4 vf = { w0.x, w0.y, w1.x, w1.y };
            if (care)
            {
                const u32x4 ind = take_nonfinite<IO>(vf);
                #pragma unroll
                for (int n = 0; n < NC; ++n)
                {
                    const f32x4 c = mfma16<IO>(ind, see[n], f32x4{});
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][t][e] += nonfinite_sum(c[e]);
                }
            }
            #pragma unroll
            for (int n = 0; n < NC; ++n) o[n][t] = mfma16<IO>(vf, pf[n], o[n][t]);
        }
    }
    // Join the waves: o against the common maximum, through LDS as [row][HD] floats with the 16-byte chunks of a
    // row permuted by its low bits.
    float lw[NC];
    #pragma unroll
    for (int n = 0; n < NC; ++n)
    {
        lw[n] = sum_xor32(sum_xor16(l[n]));
        if (quad == 0) { mlw[wave][0][16 * n + col] = m[n]; mlw[wave][1][16 * n + col] = lw[n]; }
    }
    __syncthreads();
    #pragma unroll
    for (int n = 0; n < NC; ++n)
    {
        const int r = 16 * n + col;
        float mm = -INFINITY;
        #pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, mlw[w][0][r]);
        const float ref = (mm == -INFINITY ? 0.0f : mm) * a.c;
        const float f = __builtin_amdgcn_exp2f(fmaf(m[n], a.c, -ref));
        #pragma unroll
        for (int t = 0; t < HD / 16; ++t)
        {
            f32x4 w;
            #pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = lw[n] != 0.0f ? o[n][t][e] * f : 0.0f;
            *(f32x4*)(kl + r * (HD * 4) + (((4 * t + quad) ^ (col & 7)) << 4)) = w;
        }
    }
    __syncthreads();
    // 256 lanes walk the rows: HD / 4 lanes of four columns each per row.
    constexpr int LPR = HD / 4, RPS = 256 / LPR;
    const int nr = min(ROWS, a.rows - r0);
    for (int r = tid / LPR; r < nr; r += RPS)
    {
        const int ch = tid % LPR;
        f32x4 sum{};
        float mm = -INFINITY, ls = 0.0f;
        #pragma unroll
        for (int w = 0; w < 4; ++w)
        {
            const f32x4 v = *(const f32x4*)(lds[w] + r * (HD * 4) + ((ch ^ (r & 7)) << 4));
            #pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += v[e];
            mm = fmaxf(mm, mlw[w][0][r]);
        }
        const float rf = (mm == -INFINITY ? 0.0f : mm) * a.c;
        #pragma unroll
        for (int w = 0; w < 4; ++w) ls = fmaf(mlw[w][1][r], __builtin_amdgcn_exp2f(fmaf(mlw[w][0][r], a.c, -rf)), ls);
        const QRow qr = query_row(a, it.set, it.kvh, r0 + r);
        const int64_t gr = qr.tok * a.hq + qr.h;
        if (a.direct)
        {
            const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
            if (a.lse && ch == 0) a.lse[gr] = ls == 0.0f ? -INFINITY : (rf - kShift<IO> + __builtin_amdgcn_logf(ls)) * 0.69314718055994530942f;
            store_out4<IO>(a, qr.tok, qr.h, 4 * ch, sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
        }
        else
        {
            const int64_t pr = gr * a.splits + a.split0 + it.split;
            if (ch == 0) { a.pml[2 * pr] = fmaf(mm, a.c, -kShift<IO>); a.pml[2 * pr + 1] = ls; }
            if (ls != 0.0f) ((gptr<f32x4>)(a.po + pr * HD))[ch] = sum;
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Joins the splits of a row: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.  WAVES waves per row; a wave takes
// 256 / HD splits at a time (HD / 4 lanes of four columns each).
template <class IO, int HD, int WAVES>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a)
{
    constexpr int LPR = HD / 4, SPW = 64 / LPR;       // lanes per partial row, partial rows per wave
    __shared__ float wt[4 / WAVES][kMaxSplits];
    __shared__ f32x4 part[4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, local = wave / WAVES, sub = wave % WAVES;
    const int64_t gr = min((int64_t)blockIdx.x * (4 / WAVES) + local, a.rows_all - 1);
    const int ns = a.splits;
    const gcptr<f32x2> ml = (gcptr<f32x2>)(a.pml + 2 * gr * ns);
    float m = -INFINITY, l = 0.0f;
    for (int i = lane; i < ns; i += 64)
    {
        const f32x2 e = ml[i];
        if (e.y != 0.0f) m = fmaxf(m, e.x);
    }
    m = max_wave(m);
    for (int i = lane; i < ns; i += 64)
    {
        const f32x2 e = ml[i];
        const float w = e.y != 0.0f ? __builtin_amdgcn_exp2f(e.x - (m == -INFINITY ? 0.0f : m)) : 0.0f;
        if (sub == 0) wt[local][i] = e.y != 0.0f ? w : -1.0f;      // -1: nothing was written
        if (e.y != 0.0f) l = fmaf(w, e.y, l);
    }
    l = group_sum<64>(l);
    __syncthreads();
    f32x4 o{};
    const gcptr<f32x4> po = (gcptr<f32x4>)(a.po + gr * ns * HD) + lane % LPR;
    #pragma unroll 4
    for (int i = sub * SPW + lane / LPR; i < ns; i += WAVES * SPW)
    {
        const float w = wt[local][i];
        if (w < 0.0f) continue;
        const f32x4 p = po[(int64_t)i * LPR];
        #pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(w, p[e], o[e]);
    }
    part[wave][lane] = o;
    __syncthreads();
    if (sub != 0 || lane >= LPR || (int64_t)blockIdx.x * (4 / WAVES) + local >= a.rows_all) return;
    #pragma unroll
    for (int w = 0; w < WAVES; ++w)
        #pragma unroll
        for (int k = 0; k < SPW; ++k)
        {
            if (w == 0 && k == 0) continue;
            const f32x4 p = part[local * WAVES + w][k * LPR + lane];
            #pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += p[e];
        }
    const int64_t tok = gr / a.hq;
    const int h = (int)(gr - tok * a.hq);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (a.lse && lane == 0) a.lse[gr] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.69314718055994530942f;
    store_out4<IO>(a, tok, h, 4 * lane, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

}  // namespace exl3r

using namespace exl3r;

namespace {

struct Phase
{
    int cols;       // 0: k_attn_rows; 1, 2: k_attn_keys with that many column tiles
    int64_t sets, rows, row_tiles, nsplit;
};

// How a phase is cut: `sets` row sets of `rows` query rows per KV head against at most `span` keys.
Phase plan_phase(int64_t sets, int64_t rows, int hk, int64_t span)
{
    Phase p;
    p.cols = rows <= 16 ? 1 : rows <= 32 ? 2 : 0;
    p.sets = sets;
    p.rows = rows;
    const int64_t per_tile = p.cols ? 16 * p.cols : 128;
    p.row_tiles = (rows + per_tile - 1) / per_tile;
    const int64_t base = sets * hk * p.row_tiles;
    const int64_t want = p.cols ? 4096 : 512, least = p.cols ? 128 : 256;
    int64_t n = (want + base - 1) / base;
    const int64_t most = (span + least - 1) / least;
    if (n > most) n = most;
    if (n > kMaxSplits / 2) n = kMaxSplits / 2;
    p.nsplit = n < 1 ? 1 : n;
    return p;
}

struct Plan
{
    Phase prefix, own;      // prefix.nsplit 0: none
    int64_t splits;
    bool join;
    size_t bytes;
};

Plan make_plan(int64_t bsz, int64_t seq, int hq, int hk, int hd, int64_t cap, int64_t window, int64_t sinks, int64_t shared)
{
    Plan p{};
    const int64_t group = hq / hk;
    int64_t span = cap - shared;
    if (window > 0)
    {
        const int64_t w = window + seq + sinks + 256;
        if (w < span) span = w;
    }
    p.own = plan_phase(bsz, seq * group, hk, span);
    if (shared > 0) p.prefix = plan_phase(1, bsz * seq * group, hk, shared);
    p.splits = p.own.nsplit + p.prefix.nsplit;
    p.join = p.splits > 1;
    if (p.join) p.bytes = ((size_t)p.splits * (size_t)(bsz * seq * hq) * (size_t)(hd + 2) * 4 + 255) & ~(size_t)255;
    return p;
}

int attn_entry(const char* op, const void* q, int64_t q_ts, int64_t q_hs, int hq, const void* kc, const void* vc, int hk,
               int page_size, int64_t num_pages, const int32_t* table, int64_t max_blocks, const int32_t* lens, int dtype,
               int64_t bsz, int64_t seq, int hd, int64_t shared, float scale, int window, int sinks, void* out,
               int64_t o_ts, int64_t o_hs, float* lse, int32_t* err, void* ws, size_t ws_bytes, void* stream)
{
    if (dtype != EXL3R_F16 && dtype != EXL3R_BF16)
        return set_error(EXL3R_EDTYPE, "%s: dtype must be f16 or bf16, not %s", op, dtype_name(dtype));
    if (hd != 64 && hd != 128 && hd != 256) return set_error(EXL3R_EINVAL, "%s: head_dim %d is not 64, 128 or 256", op, hd);
    if (bsz < 0 || seq < 0 || hq <= 0 || hk <= 0 || hq % hk)
        return set_error(EXL3R_EINVAL, "%s: invalid shape bsz=%lld seq_len=%lld heads %d / %d", op, (long long)bsz, (long long)seq, hq, hk);
    if (page_size <= 0 || (page_size & (page_size - 1)))
        return set_error(EXL3R_EINVAL, "%s: page_size %d is not a power of two", op, page_size);
    if (num_pages <= 0 || num_pages > 0x7fffffffLL || max_blocks <= 0)
        return set_error(EXL3R_EINVAL, "%s: invalid cache num_pages=%lld max_blocks_per_seq=%lld", op, (long long)num_pages, (long long)max_blocks);
    if (!(scale > 0.0f) || scale > 3.0e38f) return set_error(EXL3R_EINVAL, "%s: scale must be positive and finite", op);
    if (sinks < 0 || (window <= 0 && sinks != 0))
        return set_error(EXL3R_EINVAL, "%s: sinks (%d) must be 0 or more, and 0 without a window", op, sinks);
    if (bsz == 0 || seq == 0) return EXL3R_OK;
    const int64_t group = hq / hk;
    if (max_blocks > 0x7fffffc0LL / page_size || bsz > 0x7fffffffLL || seq > 0x7fffffffLL || bsz * seq > 0x7fffffffLL / hq)
        return set_error(EXL3R_EINVAL, "%s: more than 2^31 positions or query rows", op);
    const int64_t cap = max_blocks * page_size;
    if (window >= cap) window = sinks = 0;      // every position of the table is inside
    if (shared < 0 || shared % page_size || shared > cap)
        return set_error(EXL3R_EINVAL, "%s: shared_len %lld is not a whole number of the table's pages", op, (long long)shared);
    if (!q || !kc || !vc || !table || !lens || !out)
        return set_error(EXL3R_EINVAL, "%s: q, caches, block_table, cache_seqlens and out must be non-null", op);
    if (!aligned16(kc) || !aligned16(vc)) return set_error(EXL3R_EINVAL, "%s: the caches must be 16-byte aligned", op);
    const int64_t tokens = bsz * seq;
    if ((hq > 1 && (q_hs < hd || o_hs < hd)) || (tokens > 1 && (q_ts < hd || o_ts < hd)))
        return set_error(EXL3R_EINVAL, "%s: strides shorter than a head", op);
    const Plan p = make_plan(bsz, seq, hq, hk, hd, cap, window, sinks, shared);
    if (p.own.sets * hk * p.own.row_tiles * p.own.nsplit > 0xffffff || p.prefix.sets * hk * p.prefix.row_tiles * p.prefix.nsplit > 0xffffff ||
        (p.join && tokens * hq > 0xffffff))
        return set_error(EXL3R_EINVAL, "%s: more than 2^24 workgroups", op);
    if (p.join && (!ws || ((uintptr_t)ws & 255) || ws_bytes < p.bytes))
        return set_error(EXL3R_EINVAL, "%s: the workspace must be 256-byte aligned and hold %zu bytes (%zu given)", op, p.bytes, ws ? ws_bytes : 0);

    AttnArgs a{};
    a.q = (const char*)q;
    a.out = (char*)out;
    a.lse = lse;
    a.kc = (const char*)kc;
    a.vc = (const char*)vc;
    a.table = table;
    a.lens = lens;
    a.err = err;
    a.rows_all = tokens * hq;
    a.po = (float*)ws;
    a.splits = (int)p.splits;
    a.pml = p.join ? (float*)ws + p.splits * a.rows_all * hd : nullptr;
    a.q_ts = q_ts; a.q_hs = q_hs; a.o_ts = o_ts; a.o_hs = o_hs;
    a.max_blocks = max_blocks;
    a.num_pages = num_pages;
    a.bsz = (int)bsz; a.seq = (int)seq; a.hq = hq; a.hk = hk; a.group = (int)group;
    a.page_shift = __builtin_ctz((unsigned)page_size);
    a.window = window > 0 ? window : 0;
    a.sinks = sinks;
    a.direct = !p.join;
    a.q_vec = aligned16(q) && (hq == 1 || q_hs % 8 == 0) && (tokens == 1 || q_ts % 8 == 0);
    a.o_vec = ((uintptr_t)out & 7) == 0 && (hq == 1 || o_hs % 4 == 0) && (tokens == 1 || o_ts % 4 == 0);
    a.c = scale * 1.4426950408889634f;
    hipStream_t st = (hipStream_t)stream;

    auto run = [&](auto T, auto HDC) {
        using IO = decltype(T);
        constexpr int HD = decltype(HDC)::value;
        auto phase = [&](const Phase& ph, bool whole, int64_t lo, int64_t hi, int64_t split0) {
            AttnArgs x = a;
            x.whole = whole;
            x.dom_lo = (int)lo;
            x.dom_hi = (int)hi;
            x.rows = (int)ph.rows;
            x.row_tiles = (int)ph.row_tiles;
            x.nsplit = (int)ph.nsplit;
            x.split0 = (int)split0;
            const int64_t grid = ph.sets * hk * ph.row_tiles * ph.nsplit;
            if (ph.cols == 0)
            {
                if (page_size < 64) launch(k_attn_rows<IO, HD, 1, true>, (unsigned)grid, 256, 0, st, x);
                else launch(k_attn_rows<IO, HD, 1, false>, (unsigned)grid, 256, 0, st, x);
            }
            else if (ph.cols == 1)
            {
                if (page_size < 32) launch(k_attn_keys<IO, HD, 1, true>, (unsigned)grid, 256, 0, st, x);
                else launch(k_attn_keys<IO, HD, 1, false>, (unsigned)grid, 256, 0, st, x);
            }
            else
            {
                if (page_size < 32) launch(k_attn_keys<IO, HD, 2, true>, (unsigned)grid, 256, 0, st, x);
                else launch(k_attn_keys<IO, HD, 2, false>, (unsigned)grid, 256, 0, st, x);
            }
        };
        if (shared > 0) phase(p.prefix, true, 0, shared, 0);
        phase(p.own, false, shared, cap, p.prefix.nsplit);
        if (p.join)
        {
            if (p.splits > 16) launch(k_attn_join<IO, HD, 4>, (unsigned)a.rows_all, 256, 0, st, a);
            else launch(k_attn_join<IO, HD, 1>, (unsigned)((a.rows_all + 3) / 4), 256, 0, st, a);
        }
    };
    auto by_dim = [&](auto T) {
        if (hd == 64) run(T, std::integral_constant<int, 64>{});
        else if (hd == 128) run(T, std::integral_constant<int, 128>{});
        else run(T, std::integral_constant<int, 256>{});
    };
    if (dtype == EXL3R_F16) by_dim(TF16{});
    else by_dim(TBF16{});
    return launch_status(op);
}

}  // namespace

extern "C" size_t exl3r_paged_attn_workspace_bytes(int64_t bsz, int64_t seq_len, int num_heads_q, int num_heads_kv,
                                                   int head_dim, int page_size, int64_t max_blocks_per_seq, int64_t shared_len)
{
    if (bsz <= 0 || seq_len <= 0 || num_heads_q <= 0 || num_heads_kv <= 0 || head_dim <= 0 || page_size <= 0 ||
        max_blocks_per_seq <= 0 || max_blocks_per_seq > 0x7fffffffLL / page_size || bsz > 0x7fffffffLL || seq_len > 0x7fffffffLL ||
        bsz * seq_len > 0x7fffffffLL / num_heads_q || num_heads_q % num_heads_kv || shared_len < 0 ||
        shared_len > max_blocks_per_seq * page_size)
        return 0;
    return make_plan(bsz, seq_len, num_heads_q, num_heads_kv, head_dim, max_blocks_per_seq * page_size, 0, 0, shared_len).bytes;
}

extern "C" int exl3r_paged_attn(const void* q, int64_t q_tok_stride, int64_t q_head_stride, int num_heads_q,
                                const void* k_cache, const void* v_cache, int num_heads_kv, int page_size, int64_t num_pages,
                                const int32_t* block_table, int64_t max_blocks_per_seq, const int32_t* cache_seqlens,
                                int dtype, int64_t bsz, int64_t seq_len, int head_dim, float scale, int window, int sinks,
                                void* out, int64_t out_tok_stride, int64_t out_head_stride, float* lse, int32_t* err_flag,
                                void* workspace, size_t workspace_bytes, void* stream)
{
    begin_call();
    return attn_entry("exl3r_paged_attn", q, q_tok_stride, q_head_stride, num_heads_q, k_cache, v_cache, num_heads_kv,
                      page_size, num_pages, block_table, max_blocks_per_seq, cache_seqlens, dtype, bsz, seq_len, head_dim, 0,
                      scale, window, sinks, out, out_tok_stride, out_head_stride, lse, err_flag, workspace, workspace_bytes,
                      stream);
}

extern "C" int exl3r_paged_attn_shared(const void* q, int64_t q_tok_stride, int64_t q_head_stride, int num_heads_q,
                                       const void* k_cache, const void* v_cache, int num_heads_kv, int page_size,
                                       int64_t num_pages, const int32_t* block_table, int64_t max_blocks_per_seq,
                                       const int32_t* cache_seqlens, int64_t shared_len, int dtype, int64_t bsz,
                                       int64_t seq_len, int head_dim, float scale, int window, int sinks, void* out,
                                       int64_t out_tok_stride, int64_t out_head_stride, float* lse, int32_t* err_flag,
                                       void* workspace, size_t workspace_bytes, void* stream)
{
    begin_call();
    return attn_entry("exl3r_paged_attn_shared", q, q_tok_stride, q_head_stride, num_heads_q, k_cache, v_cache, num_heads_kv,
                      page_size, num_pages, block_table, max_blocks_per_seq, cache_seqlens, dtype, bsz, seq_len, head_dim,
                      shared_len, scale, window, sinks, out, out_tok_stride, out_head_stride, lse, err_flag, workspace,
                      workspace_bytes, stream);
}
