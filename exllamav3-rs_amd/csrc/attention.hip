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
#include <algorithm>
#include "abi.hpp"
#include "common.cuh"

namespace exl3r {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <class T> using lptr = __attribute__((address_space(3))) T*;

constexpr int kMaxSplits = 512;      // of a row in one launch

// Where a launch leaves the partial results of its rows: o unnormalised, {c m - shift, l}, fp32.  Partial i of a row:
//   k_attn_rows: of `n` fixed splits, at [global row][i];
//   k_attn_keys (`info` set): of the workgroups ("slots") info[seg].x .. info[seg].y that share its segment, at
//   [KV head][slot + seg][row of the segment]: slot + seg never meets itself, as walking the slots one or the other
//   grows.
struct Parts
{
    float* po;
    float* ml;
    int32_t* info;
    int32_t n, slots, segs, row_tiles, seg_rows, whole;
};

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
    Parts parts;              // of this launch
    int64_t q_ts, q_hs, o_ts, o_hs;     // elements
    int64_t max_blocks, num_pages;
    int64_t rows_all;         // bsz * seq * hq
    int32_t bsz, seq, hq, hk, group;
    int32_t page_shift, window, sinks;
    int32_t dom_lo, dom_hi;   // keys of this launch: [dom_lo, dom_hi)
    int32_t rows;             // query rows per row set (a sequence's, or the whole batch's)
    int32_t row_tiles;
    int32_t whole;            // 1: one row set of all sequences, keys through sequence 0's table row
    int32_t direct;           // 1: a result that no other split shares is the output
    int32_t q_vec, o_vec;     // 16-byte aligned q rows / 8-byte aligned out rows
    float c;
};

constexpr float kLn2 = 0.69314718055994530942f;

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
__device__ __forceinline__ float load_bits(uint16_t h)
{
    if constexpr (IO::code == DT_F16) return (float)__builtin_bit_cast(_Float16, h);
    else return bf16lo(h);
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

// LDS rows of a tile of K or V are HD elements and a pad that spreads what one read touches over the banks (256 bytes):
// a K read takes the same 16 bytes of 16 rows, so 16 bytes of pad; a transposing V read takes 64 bytes of 4 rows (MFMA
// tiles of 32) or 32 bytes of 8 (tiles of 16), so pads of 64 or 32.  Every address is then one register and an offset
// in the instruction, which an XOR of the chunk index, as free of conflicts, is not.
template <int HD> constexpr int kRowK = HD * 2 + 16;
template <int HD, int COLS> constexpr int kRowV = HD * 2 + 2 * COLS;

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

__device__ __forceinline__ int64_t uniform64(int64_t v)
{
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
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

// K fragment of 32 keys (LDS rows from kb on) and 16 dimensions (16 t on).
template <int HD>
__device__ __forceinline__ u32x4 k_fragment(const char* kb, int lane, int t)
{
    return *(const u32x4*)(kb + (lane & 31) * kRowK<HD> + (lane >> 5) * 16 + t * 32);
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

// The reference m of a row's exponents is its running maximum, but one that a tile exceeds by less than 2^kSlack stays:
// o and l are then not rescaled (64 of 185 VALU instructions per tile of 32 keys and 32 rows of 128, where most
// tiles raise some row's maximum a little).  Exponents are raised by kShift: as f16, whose largest number is below 2^16
// and smallest normal one 2^-14, a probability then keeps its 11 bits from 2^kSlack of the reference down to 2^-20 of
// it (bf16 has fp32's range).  o and l carry the same factor.
constexpr float kSlack = 8.0f;
template <class IO> constexpr float kShift = IO::code == DT_F16 ? 6.0f : 0.0f;

// The factor of o and l when the reference goes from m to mn, and the exponents' constant.
__device__ __forceinline__ float rescale_factor(float m, float mn, float c)
{
    return __builtin_amdgcn_exp2f((m - (mn == -INFINITY ? 0.0f : mn)) * c);
}
template <class IO> __device__ __forceinline__ float exponent_base(float m, float c)
{
    return kShift<IO> - (m == -INFINITY ? 0.0f : m) * c;
}

// V^T fragment of 16 keys (half u of the 32 at vb) and 32 columns (32 t on).
template <int HD>
__device__ __forceinline__ u32x4 v_fragment(const char* vb, int lane, int u, int t)
{
    constexpr int RV = kRowV<HD, 32>;
    const char* r0 = vb + (4 * (lane >> 5) + ((lane >> 2) & 3)) * RV + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    const auto v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr<s16x4>)(r0 + u * 16 * RV + t * 64));
    const auto v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr<s16x4>)(r0 + (u * 16 + 8) * RV + t * 64));
    const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
    return u32x4{ w0.x, w0.y, w1.x, w1.y };
}

// Infinities and NaNs of V in a tile that some row does not see whole: there the probability is 0, but 0 * inf and
// 0 * NaN must not reach the row.  They are zeroed on their way into LDS, and a workgroup that met one (rare: a bad
// activation in the cache) adds them at its end, key by key, to the rows that see them.
template <class IO>
__device__ __forceinline__ bool nonfinite(uint32_t h)     // 16 bits
{
    constexpr uint32_t E = IO::code == DT_F16 ? 0x7c00u : 0x7f80u;
    return (h & E) == E;
}
// Whether some of 8 elements is one.
template <class IO>
__device__ __forceinline__ bool nonfinite8(const u32x4& v)
{
    constexpr uint32_t E = IO::code == DT_F16 ? 0x7c00u : 0x7f80u, E2 = E | E << 16, B = E & (0u - E), B2 = B | B << 16;
    uint32_t c = 0;     // the carry of exponent + 1 out of the exponent's field: all ones there
    #pragma unroll
    for (int i = 0; i < 4; ++i) c |= ((v[i] & E2) + B2) & 0x80008000u;
    return c != 0;
}
template <class IO>
__device__ __forceinline__ void zero_nonfinite(u32x4& v)
{
    #pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] &= (nonfinite<IO>(v[i]) ? 0u : 0xffffu) | (nonfinite<IO>(v[i] >> 16) ? 0u : 0xffff0000u);
}

// The page of key j, of the last key past the end.
__device__ __forceinline__ int page_entry(const AttnArgs& a, const int32_t* table, int j, int khi)
{
    return ((gcptr<int32_t>)table)[min(j, khi - 1) >> a.page_shift];
}

// One tile's loads.  SMALL (pages of fewer keys than a tile): a lane's key has a page of its own, entry k of the
// tile's page list being in lane k.  Otherwise the tile lies in one page, at a wave-uniform base, and the keys past
// the last one are read too (they are in the page) and taken out later.  A bad page's keys read page 0.
template <int HD, bool SMALL, int STEPS, int LANES>
__device__ __forceinline__ void load_tile(const AttnArgs& a, int j0, int entry, uint64_t ok, int kvh, int lane_of_tile,
                                          u32x4 (&ks)[STEPS], u32x4 (&vs)[STEPS])
{
    constexpr int CH = HD / 8, KPS = LANES / CH;      // keys per step
    int key0 = lane_of_tile / CH, ch = lane_of_tile % CH;
    const uint32_t row_bytes = (uint32_t)a.hk * (HD * 2);
    const int in_page = (1 << a.page_shift) - 1;
    if constexpr (SMALL)
    {
        // (decode: the steps' addresses are not kept in registers from tile to tile)
        if constexpr (LANES == 64) asm volatile("" : "+v"(key0), "+v"(ch));
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

// A tile in registers of which not every row sees all: its keys that the launch must not see become zeros, V's infinities
// and NaNs too.  Returns whether there were such.
template <class IO, int HD, int STEPS, int LANES>
__device__ __forceinline__ bool clean_tile(u32x4 (&ks)[STEPS], u32x4 (&vs)[STEPS], uint64_t ok, int lane_of_tile)
{
    constexpr int CH = HD / 8, KPS = LANES / CH;
    bool odd = false;
    #pragma unroll
    for (int k = 0; k < STEPS; ++k)
    {
        if (!((ok >> (k * KPS + lane_of_tile / CH)) & 1)) ks[k] = vs[k] = u32x4{};
        if (nonfinite8<IO>(vs[k]))
        {
            zero_nonfinite<IO>(vs[k]);
            odd = true;
        }
    }
    return odd;
}

// Step k of a tile in registers, or all of it, into LDS.
template <int HD, int STEPS, int LANES, int RV>
__device__ __forceinline__ void write_step(const u32x4 (&ks)[STEPS], const u32x4 (&vs)[STEPS], int k, int lane_of_tile, char* kl, char* vl)
{
    constexpr int CH = HD / 8, KPS = LANES / CH;
    const int key = lane_of_tile / CH, ch = lane_of_tile % CH;
    *(u32x4*)(kl + key * kRowK<HD> + ch * 16 + k * KPS * kRowK<HD>) = ks[k];
    *(u32x4*)(vl + key * RV + ch * 16 + k * KPS * RV) = vs[k];
}
template <int HD, int STEPS, int LANES, int RV>
__device__ __forceinline__ void write_tile(const u32x4 (&ks)[STEPS], const u32x4 (&vs)[STEPS], int lane_of_tile, char* kl, char* vl)
{
    #pragma unroll
    for (int k = 0; k < STEPS; ++k) write_step<HD, STEPS, LANES, RV>(ks, vs, k, lane_of_tile, kl, vl);
}

// Calls add(j, v) for every key j of the tile at j0 with V's row there (global memory).
template <int HD, class F>
__device__ __forceinline__ void each_value_row(const AttnArgs& a, const TileList& l, const int32_t* table, int j0, int keys, int kvh, F&& add)
{
    for (int j = j0; j < j0 + keys && j < l.khi; ++j)
    {
        const int page = table[j >> a.page_shift];
        if ((uint64_t)(int64_t)page >= (uint64_t)a.num_pages) continue;
        const int64_t row = ((int64_t)page << a.page_shift) + (j & ((1 << a.page_shift) - 1));
        add(j, (gcptr<uint16_t>)a.vc + (row * a.hk + kvh) * HD);
    }
}
__device__ __forceinline__ bool row_sees(const AttnArgs& a, int p, int j)
{
    return j <= p && (a.window <= 0 || p - j < a.window || j < a.sinks);
}
// Whether every row with a position in [pmin, pmax] sees all of the keys j .. j + n - 1.
__device__ __forceinline__ bool all_seen(const AttnArgs& a, int j, int n, int pmin, int pmax)
{
    return j + n - 1 <= pmin && (a.window <= 0 || pmax - j < a.window || j + n - 1 < a.sinks);
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
    it.split = x % (uint32_t)a.parts.n;
    it.set = x / (uint32_t)a.parts.n;
    return it;
}

__device__ __forceinline__ void flag_positions(const AttnArgs& a, int p)
{
    const int64_t cap = a.max_blocks << a.page_shift;
    if (a.err && (p < 0 || p >= cap)) *a.err = 1;
}

// ---------------------------------------------------------------------------------------------
// Many query rows: WAVES waves of 32 rows each share tiles of KT keys in a ring of three LDS stages.  A wave's step is a
// slot of products (o += V(i) P(i), then the scores of tile i + 1) and a slot of softmax (those scores to P(i + 1), and
// its part of a later tile's loads and LDS writes), with a barrier after each.  Of 8 waves, 4 .. 7 (the second wave of
// each SIMD) run one slot behind 0 .. 3, so that one wave of a SIMD is at the matrix cores while the other is at the
// VALU: in step, both wait for the same unit.
// 256 rows and tiles of 64 keys: 113 KB of LDS and 242 registers, one workgroup per CU.  Every byte of K and V read from
// LDS then feeds 32 rows and every byte from the L2 256; rows of 128 in two workgroups per CU took 341 us for 295.
// Measured: 4096 tokens of 64 heads of 128 on 8 KV heads, bf16, 295 us, 930 TFLOP/s of the visible half.  Bound by the
// softmax's slot: of the ~4390 cycles of a tile the products of both waves take 2 x 1320, and a softmax (1230), its loads
// and LDS writes (820) and two barriers are longer than the other wave's products: the matrix cores are busy for 45% of
// a CU's time.
// Heads of 256 have o and Q of 32 rows in 192 registers: one wave per SIMD, 128 rows, tiles of 32, and products and softmax
// of the same wave interleaved, two tiles of loads under way (4 x 4096 tokens of 16 heads on 2, bf16: 712 us, 773 TFLOP/s;
// with one tile 733, products and softmax in turn 783).  Pages of 16 keys cost it the lookup of every row: 803 us.
template <class IO, int HD, int WAVES, int KT, bool SMALL>
__global__ __launch_bounds__(WAVES * 64, HD == 256 ? 1 : 2) void k_attn_rows(AttnArgs a)
{
    constexpr int LANES = WAVES * 64, RK = kRowK<HD>, RV = kRowV<HD, 32>, STEPS = KT * (HD / 8) / LANES, NS = KT / 32;
    constexpr int STAGE = KT * (RK + RV);
    constexpr uint64_t FULL = KT == 64 ? ~0ull : 0xffffffffull;
    __shared__ __align__(16) char lds[3 * STAGE];
    __shared__ int plo[WAVES], phi[WAVES], odd;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int late = WAVES == 8 ? wave >> 2 : 0;
    const Item it = launch_item(a);
    const int r0 = it.tile * (32 * WAVES) + wave * 32;
    const QRow row = query_row(a, it.set, it.kvh, min(r0 + (lane & 31), a.rows - 1));
    if (it.split == 0 && it.kvh == 0) flag_positions(a, row.p);
    const int pmin = wave_min(row.p), pmax = wave_max(row.p);
    if (lane == 0) { plo[wave] = pmin; phi[wave] = pmax; }
    if (tid == 0) odd = 0;
    u32x4 qf[HD / 16];
    load_q<IO, HD, 16>(a, row, half, qf);
    __syncthreads();
    int gmin = plo[0], gmax = phi[0];       // positions of the workgroup's rows
    #pragma unroll
    for (int w = 1; w < WAVES; ++w) { gmin = min(gmin, plo[w]); gmax = max(gmax, phi[w]); }
    gmin = __builtin_amdgcn_readfirstlane(gmin);
    gmax = __builtin_amdgcn_readfirstlane(gmax);
    const TileList tl = tile_list(a, gmin, gmax, KT);
    const int per = (tl.count + a.parts.n - 1) / a.parts.n;
    const int t0 = min(it.split * per, tl.count), t1 = min(t0 + per, tl.count);
    const int32_t* table = a.table + (a.whole ? 0 : (int64_t)it.set * a.max_blocks);
    const auto tile_key = [&](int i) { return a.dom_lo + tl.tile(i) * KT; };

    f32x16 o[HD / 32];
    #pragma unroll
    for (int t = 0; t < HD / 32; ++t) o[t] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    const float slack = fminf(kSlack / a.c, 1e38f);
    f32x16 s[NS];
    u32x4 pf[2 * NS];       // P of 16 keys each
    const auto softmax = [&](int i, uint64_t ok, bool part) {
        if (part)
        {
            const int j0 = tile_key(i);
            #pragma unroll
            for (int k = 0; k < NS; ++k)
                mask_tile(s[k], j0 + 32 * k, half, row.p, a.window, a.sinks, (uint32_t)(ok >> (32 * k)));
        }
        float mx4[4] = { s[0][0], s[0][1], s[0][2], s[0][3] };
        #pragma unroll
        for (int k = 0; k < NS; ++k)
            #pragma unroll
            for (int e = k ? 0 : 4; e < 16; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], s[k][e]);
        const float mx = max_xor32(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])));
        if (__any(mx > m + slack))
        {
            const float mn = fmaxf(m, mx), alpha = rescale_factor(m, mn, a.c);
            l *= alpha;
            m = mn;
            #pragma unroll
            for (int t = 0; t < HD / 32; ++t)
                #pragma unroll
                for (int e = 0; e < 16; ++e) o[t][e] *= alpha;
        }
        const float base = exponent_base<IO>(m, a.c);
        float sum[4] = {};
        #pragma unroll
        for (int k = 0; k < NS; ++k)
        {
            #pragma unroll
            for (int e = 0; e < 16; ++e)
            {
                s[k][e] = __builtin_amdgcn_exp2f(fmaf(s[k][e], a.c, base));
                sum[e & 3] += s[k][e];
            }
            #pragma unroll
            for (int e = 0; e < 8; ++e) pf[2 * k + e / 4][e % 4] = pack2<IO>(s[k][2 * e], s[k][2 * e + 1]);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    };

    if (t0 < t1)
    {
        // The tiles of the list that every row of the workgroup, or of the wave, sees whole: [f0, gf1) and [f0 or its own,
        // wf1) (the sinks' tiles aside).
        const auto whole_from = [&](int pmx) { return a.window > 0 ? max(tl.ns, tl.ns - tl.wt + (max(max(pmx - a.window + 1, 0) - a.dom_lo, 0) + KT - 1) / KT) : tl.ns; };
        const auto whole_to = [&](int pmn) { return tl.ns - tl.wt + max(min(pmn, 0x7ffffffe) + 1 - a.dom_lo, 0) / KT; };
        const int gf0 = whole_from(gmax), gf1 = whole_to(gmin), wf0 = whole_from(pmax), wf1 = whole_to(pmin);

        // Loads.  SMALL: every key's page is looked up.  Otherwise a tile lies in one page and follows the one before it,
        // but for the step from the sinks to the window; `off` is its first row's byte offset for this KV head.  Past the
        // last tile the last one is loaded again.
        u32x4 ks[STEPS], vs[STEPS];
        const uint32_t row_bytes = (uint32_t)a.hk * (HD * 2);
        const int in_page = (1 << a.page_shift) - 1, last_page = (tl.khi - 1) >> a.page_shift;
        uint64_t ok0 = 0, ok1 = 0, ok2 = 0, ok3 = 0;      // the visible keys of the last tiles loaded that have a page
        bool bad = false;
        int entry = 0, ahead = 0, il = t0;       // (SMALL: a key's page each) page of tile il, of the page after it
        int64_t off = 0;
        const auto enter_page = [&](int j, int e) {      // tile il starts at key j of page e
            const bool good = (uint32_t)e < (uint32_t)a.num_pages;
            bad |= !good;
            entry = good;
            off = ((int64_t)(good ? e : 0) << a.page_shift) + (j & in_page);
            off = off * row_bytes + it.kvh * (HD * 2);
            ahead = ((gcptr<int32_t>)table)[min((j >> a.page_shift) + 1, last_page)];
        };
        if constexpr (SMALL) entry = page_entry(a, table, tile_key(t0) + (lane & (KT - 1)), tl.khi);
        else enter_page(tile_key(t0), __builtin_amdgcn_readfirstlane(((gcptr<int32_t>)table)[tile_key(t0) >> a.page_shift]));
        const uint32_t lane_off = tid / (HD / 8) * row_bytes + tid % (HD / 8) * 16;
        const auto load_into = [&](u32x4 (&ks)[STEPS], u32x4 (&vs)[STEPS]) __attribute__((always_inline)) {
            ok3 = ok2;
            ok2 = ok1;
            ok1 = ok0;
            if constexpr (SMALL)
            {
                const int j0 = tile_key(il);
                const bool in = key_seen(a, tl, j0 + (lane & (KT - 1)), gmin), good = in && (uint32_t)entry < (uint32_t)a.num_pages;
                bad |= in && !good;
                ok0 = __ballot(good) & FULL;
                load_tile<HD, SMALL, STEPS, LANES>(a, j0, entry, ok0, it.kvh, tid, ks, vs);
                if (il + 1 < t1) ++il;
                entry = page_entry(a, table, tile_key(il) + (lane & (KT - 1)), tl.khi);
            }
            else
            {
                ok0 = entry ? FULL : 0;
                const char *kb = a.kc + off, *vb = a.vc + off;
                #pragma unroll
                for (int k = 0; k < STEPS; ++k)
                {
                    ks[k] = *(gcptr<u32x4>)(kb + lane_off);
                    vs[k] = *(gcptr<u32x4>)(vb + lane_off);
                    kb += LANES / (HD / 8) * row_bytes;
                    vb += LANES / (HD / 8) * row_bytes;
                }
                if (il + 1 < t1)
                {
                    ++il;
                    const int j = tile_key(il);
                    if (il == tl.ns) enter_page(j, __builtin_amdgcn_readfirstlane(((gcptr<int32_t>)table)[j >> a.page_shift]));
                    else if ((j & in_page) == 0) enter_page(j, __builtin_amdgcn_readfirstlane(ahead));
                    else off += KT * row_bytes;
                }
            }
        };
        // The tile loaded last, tile i, into stage st: clean where not every row sees all of it.
        const auto load = [&]() { load_into(ks, vs); };
        const auto clean = [&](int i, u32x4 (&ks)[STEPS], u32x4 (&vs)[STEPS], uint64_t ok) {
            i = min(i, t1 - 1);
            if (i < gf0 || i >= gf1 || ok != FULL)
            {
                uint64_t seen = ok;
                if (!SMALL) seen &= __ballot(key_seen(a, tl, tile_key(i) + (lane & (KT - 1)), gmin));
                if (clean_tile<IO, HD, STEPS, LANES>(ks, vs, seen, tid)) odd = 1;
            }
        };
        const auto write = [&](int i, char* st) {
            clean(i, ks, vs, ok0);
            write_tile<HD, STEPS, LANES, RV>(ks, vs, tid, st, st + KT * RK);
        };

        if constexpr (WAVES == 4)
        {
            // One wave per SIMD: its own products and softmax overlap.  A step multiplies the scores of tile i + 1, with the LDS
            // writes of tile i + 2 between the MFMAs, then o += V(i) P(i) with the softmax of tile i + 1 between them: both
            // take about as long.  What raises the reference m is applied to o after that.
            static_assert(NS == 1);
            char *sa = lds, *sb = lds + STAGE, *sc = lds + 2 * STAGE;
            load();
            write(t0, sa);
            load();
            write(t0 + 1, sb);
            load();
            u32x4 kb[STEPS], vb[STEPS];     // (two tiles of loads under way)
            load_into(kb, vb);
            __syncthreads();
            constexpr int N = HD / 16, AHEAD = 8;
            #pragma unroll
            for (int j = 0; j < N; ++j) s[0] = mfma32<IO>(k_fragment<HD>(sa, lane, j), qf[j], j == 0 ? f32x16{} : s[0]);
            softmax(t0, ok3, t0 < wf0 || t0 >= wf1 || ok3 != FULL);
            const auto step = [&](int i, u32x4 (&ks)[STEPS], u32x4 (&vs)[STEPS]) __attribute__((always_inline)) {
                clean(i + 2, ks, vs, ok1);
                u32x4 f[AHEAD];
                const auto read = [&](int j) {
                    if (j < N) f[j % AHEAD] = k_fragment<HD>(sb, lane, j);
                    else f[j % AHEAD] = v_fragment<HD>(sa + KT * RK, lane, (j - N) / (HD / 32), (j - N) % (HD / 32));
                };
                #pragma unroll
                for (int j = 0; j < AHEAD; ++j) read(j);
                #pragma unroll
                for (int j = 0; j < N; ++j)
                {
                    __builtin_amdgcn_sched_barrier(0);
                    s[0] = mfma32<IO>(f[j % AHEAD], qf[j], j == 0 ? f32x16{} : s[0]);
                    read(j + AHEAD);
                    if (j >= N - STEPS) write_step<HD, STEPS, LANES, RV>(ks, vs, j - (N - STEPS), tid, sc, sc + KT * RK);
                }
                __builtin_amdgcn_sched_barrier(0);
                load_into(ks, vs);
                const bool live = i + 1 < t1;
                const uint64_t ok = live ? ok3 : 0;
                float mx4[4], sum[4] = {}, alpha = 1.0f, base = 0.0f;
                bool raised = false;
                #pragma unroll
                for (int j = 0; j < N; ++j)
                {
                    __builtin_amdgcn_sched_barrier(0);
                    o[j % (HD / 32)] = mfma32<IO>(f[(N + j) % AHEAD], pf[j / (HD / 32)], o[j % (HD / 32)]);
                    if (j + AHEAD < N) read(N + j + AHEAD);
                    if (j == 1)
                    {
                        if (!live || i + 1 < wf0 || i + 1 >= wf1 || ok != FULL)
                            mask_tile(s[0], tile_key(min(i + 1, t1 - 1)), half, row.p, a.window, a.sinks, (uint32_t)ok);
                        #pragma unroll
                        for (int e = 0; e < 8; ++e) mx4[e & 3] = e < 4 ? s[0][e] : fmaxf(mx4[e & 3], s[0][e]);
                    }
                    if (j == 2)
                    {
                        #pragma unroll
                        for (int e = 8; e < 16; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], s[0][e]);
                    }
                    if (j == 3)
                    {
                        const float mx = max_xor32(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])));
                        raised = __any(mx > m + slack);
                        const float mn = raised ? fmaxf(m, mx) : m;
                        alpha = rescale_factor(m, mn, a.c);
                        l = raised ? l * alpha : l;
                        m = mn;
                        base = exponent_base<IO>(m, a.c);
                    }
                    if (j >= 4 && j < 12)
                    {
                        #pragma unroll
                        for (int e = 2 * (j - 4); e < 2 * (j - 4) + 2; ++e)
                        {
                            s[0][e] = __builtin_amdgcn_exp2f(fmaf(s[0][e], a.c, base));
                            sum[e & 3] += s[0][e];
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                #pragma unroll
                for (int e = 0; e < 8; ++e) pf[e / 4][e % 4] = pack2<IO>(s[0][2 * e], s[0][2 * e + 1]);
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if (raised)
                {
                    #pragma unroll
                    for (int t = 0; t < HD / 32; ++t)
                        #pragma unroll
                        for (int e = 0; e < 16; ++e) o[t][e] *= alpha;
                }
                char* const st = sa;
                sa = sb;
                sb = sc;
                sc = st;
                __syncthreads();
            };
            for (int i = t0; i < t1; i += 2)
            {
                step(i, ks, vs);
                if (i + 1 < t1) step(i + 1, kb, vb);
            }
        }
        else
        {
        // A slot's products: o += V P with V of stage v (if `step`), then the scores of the keys of stage k.  LDS reads run
        // 8 MFMAs ahead of their use, in this order exactly: left to itself the compiler reads just before it
        // multiplies, and waits for each read.
        const auto products = [&](auto step, const char* v, const char* k) __attribute__((always_inline)) {
            constexpr int N = NS * HD / 16, AHEAD = 8;      // MFMAs of each product
            constexpr int from = decltype(step)::value ? 0 : N;
            u32x4 f[AHEAD];
            const auto read = [&](int j) {
                if (j < N) f[j % AHEAD] = v_fragment<HD>(v + KT * RK + j / (HD / 16) * 32 * RV, lane, j / (HD / 32) % 2, j % (HD / 32));
                else f[j % AHEAD] = k_fragment<HD>(k + (j - N) % NS * 32 * RK, lane, (j - N) / NS);
            };
            #pragma unroll
            for (int j = 0; j < AHEAD; ++j) read(from + j);
            #pragma unroll
            for (int j = from; j < 2 * N; ++j)
            {
                __builtin_amdgcn_sched_barrier(0);
                if (j < N) o[j % (HD / 32)] = mfma32<IO>(f[j % AHEAD], pf[j / (HD / 32)], o[j % (HD / 32)]);
                else s[(j - N) % NS] = mfma32<IO>(f[j % AHEAD], qf[(j - N) / NS], j - N < NS ? f32x16{} : s[(j - N) % NS]);
                if (j + AHEAD < 2 * N) read(j + AHEAD);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        const auto probabilities = [&](int i, uint64_t ok) { softmax(i, ok, i < wf0 || i >= wf1 || ok != FULL); };

        // The stages of tiles i, i + 1 and i + 2.  The late waves write, and load, a tile further: tile i + 3's stage held
        // tile i, which they are the last to read.
        char *sa = lds, *sb = lds + STAGE, *sc = lds + 2 * STAGE;
        load();
        write(t0, sa);
        load();
        write(t0 + 1, sb);
        load();
        const uint64_t first = ok2;
        if (late)
        {
            write(t0 + 2, sc);
            load();
        }
        __syncthreads();
        if (late) __syncthreads();
        products(std::false_type{}, sa, sa);
        __syncthreads();
        probabilities(t0, first);
        __syncthreads();
        for (int i = t0; i < t1; ++i)
        {
            products(std::true_type{}, sa, sb);
            __syncthreads();
            if (i + 1 < t1) probabilities(i + 1, late ? ok2 : ok1);
            write(i + 2 + late, late ? sa : sc);
            load();
            char* const st = sa;
            sa = sb;
            sb = sc;
            sc = st;
            __syncthreads();
        }
        }
        if (!late && WAVES == 8) __syncthreads();
        if (a.err && bad) *a.err = 1;
    }
    __syncthreads();
    if (odd)
        for (int i = t0; i < t1; ++i)
            each_value_row<HD>(a, tl, table, tile_key(i), KT, it.kvh, [&](int j, gcptr<uint16_t> v) {
                #pragma unroll
                for (int t = 0; t < HD / 32; ++t)
                    #pragma unroll
                    for (int e = 0; e < 16; ++e)
                    {
                        const uint16_t h = v[32 * t + 8 * (e / 4) + 4 * half + e % 4];
                        if (nonfinite<IO>(h) && row_sees(a, row.p, j)) o[t][e] += load_bits<IO>(h);
                    }
            });
    l = sum_xor32(l);
    if (r0 + (lane & 31) >= a.rows) return;
    const int64_t gr = row.tok * a.hq + row.h;
    if (a.direct)
    {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (a.lse && half == 0) a.lse[gr] = l == 0.0f ? -INFINITY : (fmaf(m, a.c, -kShift<IO>) + __builtin_amdgcn_logf(l)) * kLn2;
        #pragma unroll
        for (int t = 0; t < HD / 32; ++t)
            #pragma unroll
            for (int g = 0; g < 4; ++g)
                store_out4<IO>(a, row.tok, row.h, 32 * t + 8 * g + 4 * half, o[t][4 * g] * inv, o[t][4 * g + 1] * inv,
                               o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv);
    }
    else
    {
        const int64_t pr = gr * a.parts.n + it.split;
        if (half == 0) { a.parts.ml[2 * pr] = fmaf(m, a.c, -kShift<IO>); a.parts.ml[2 * pr + 1] = l; }
        if (l == 0.0f) return;
        gptr<f32x4> d = (gptr<f32x4>)(a.parts.po + pr * HD + 4 * half);
        #pragma unroll
        for (int t = 0; t < HD / 32; ++t)
            #pragma unroll
            for (int g = 0; g < 4; ++g)
                d[8 * t + 2 * g] = f32x4{ o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3] };
    }
}

// ---------------------------------------------------------------------------------------------
// Few query rows (decode): the 4 waves of a workgroup hold the same NC * 16 rows and walk different tiles of 32 keys,
// each through its own part of LDS without a barrier; their results are joined at the end.  With 16 rows per MFMA
// column tile (v_mfma_f32_16x16x32: lane l holds row l % 16, keys 4 (l / 16) + i of each 16) a group of 8 or 16 query
// heads leaves little of a tile empty, and o, Q and the scores take half the registers of 32 rows, so that two tiles
// of loads per SIMD stay in flight: HBM is the bound here.  Measured: 64 sequences of 700 to 8100 keys, 64 heads of 128
// on 8, f16, 208 us, 5.5 TB/s of the cache; 2 of 98765 and 131000, 32 heads on 4, 91 us, 5.4 TB/s; a copy of 1 GiB
// moves 6.6 TB/s (reads and writes).
// The work is cut by keys, not by rows: the row tiles of all sequences ("segments"), in units of 128 keys, make one
// list per KV head, and each of `slots` workgroups takes an equal part of it, whatever the lengths.  Every workgroup
// counts the units itself, from cache_seqlens; a segment that one slot has whole goes straight to the output.

// The units of segment g (never 0: its rows are written also where they see nothing).
__device__ __forceinline__ int list_units(const TileList& l) { return max(1, (l.count + 3) / 4); }

__device__ __forceinline__ int segment_units(const AttnArgs& a, int g)
{
    const int b = g / a.row_tiles, r0 = (g - b * a.row_tiles) * a.parts.seg_rows, r1 = min(r0 + a.parts.seg_rows, a.rows) - 1;
    const int64_t len = a.lens[b], lo = len + r0 / a.group, hi = len + r1 / a.group;
    return list_units(tile_list(a, (int)min(max(lo, (int64_t)-1), (int64_t)0x7fffffff),
                                (int)min(max(hi, (int64_t)-1), (int64_t)0x7fffffff), 32));
}

template <class IO, int HD, int NC, bool SMALL>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void k_attn_keys(AttnArgs a)
{
    constexpr int KT = 32, RK = kRowK<HD>, RV = kRowV<HD, 16>, STEPS = KT * (HD / 8) / 64, ROWS = 16 * NC;
    __shared__ __align__(16) char lds[4][KT * (RK + RV)];
    __shared__ float mlw[4][2][ROWS];
    __shared__ int64_t sums[4], begin[2];
    int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    char* const kl = lds[wave];
    char* const vl = lds[wave] + KT * RK;
    const int kvh = blockIdx.x % (uint32_t)a.hk, slot = blockIdx.x / (uint32_t)a.hk, segs = a.parts.segs;

    int pos[NC], set = 0, r0 = 0, pmin = 0, pmax = 0, units = 0;
    TileList tl{};
    const auto enter = [&](int g) {
        const int col = tid & 15;
        set = a.whole ? 0 : g / a.row_tiles;
        r0 = (g - set * a.row_tiles) * ROWS;
        pmin = 0x7fffffff;
        pmax = -0x7fffffff;
        #pragma unroll
        for (int n = 0; n < NC; ++n)
        {
            pos[n] = query_row(a, set, kvh, min(r0 + 16 * n + col, a.rows - 1)).p;
            pmin = min(pmin, pos[n]);
            pmax = max(pmax, pos[n]);
        }
        pmin = wave_min(pmin);
        pmax = wave_max(pmax);
        tl = tile_list(a, pmin, pmax, KT);
        units = list_units(tl);
    };
    // The slot's units [x0, x1), the segment that x0 lies in and that segment's first unit.
    int64_t total = 0, start = 0;
    int g = 0;
    if (segs == 1)
    {
        enter(0);
        total = units;
    }
    else
    {
        const int each = (segs + 255) / 256, g0 = min(tid * each, segs), g1 = min(g0 + each, segs);
        int64_t mine = 0;
        if (!a.whole)
            for (int i = g0; i < g1; ++i) mine += segment_units(a, i);
        else        // (two row tiles at most)
            for (int i = 0; i < segs; ++i)
            {
                enter(i);
                if (g0 <= i && i < g1) mine += units;
            }
        int64_t before = mine;
        #pragma unroll
        for (int d = 1; d < 64; d <<= 1)
        {
            const int64_t v = __shfl_up(before, d);
            if ((tid & 63) >= d) before += v;
        }
        if ((tid & 63) == 63) sums[wave] = before;
        __syncthreads();
        before -= mine;
        #pragma unroll
        for (int w = 0; w < 4; ++w)
        {
            if (w < wave) before += sums[w];
            total += sums[w];
        }
        const int64_t x = slot * ((total + a.parts.slots - 1) / a.parts.slots);
        if (x >= before && x < before + mine)
        {
            if (!a.whole)
                for (g = g0; ; ++g)
                {
                    const int u = segment_units(a, g);
                    if (x < before + u) break;
                    before += u;
                }
            else g = g0;        // (one segment per lane)
            begin[0] = g;
            begin[1] = before;
        }
        __syncthreads();
        g = __builtin_amdgcn_readfirstlane((int)begin[0]);
        start = uniform64(begin[1]);
        total = uniform64(total);
    }
    const int64_t share = uniform64((total + a.parts.slots - 1) / a.parts.slots), x0 = slot * share, x1 = min(x0 + share, total);
    if (x0 >= total) return;
    const float slack = fminf(kSlack / a.c, 1e38f);
    for (;; ++g)
    {
    if (segs != 1) enter(g);
    // (Pinned here and below: what a lane computes from its number would be kept across the loop over the segments, in
    // registers that the loop over the keys needs.)
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, quad = lane >> 4, col = lane & 15;
    const int u0 = (int)max(x0 - start, (int64_t)0), u1 = (int)min(x1 - start, (int64_t)units);
    const int t0 = __builtin_amdgcn_readfirstlane(min(4 * u0, tl.count)), t1 = __builtin_amdgcn_readfirstlane(min(4 * u1, tl.count));
    if (u0 == 0 && kvh == 0)
    {
        #pragma unroll
        for (int n = 0; n < NC; ++n) flag_positions(a, pos[n]);
        if (tid == 0 && a.parts.info)
        {
            a.parts.info[2 * g] = slot;
            a.parts.info[2 * g + 1] = (int)((start + units - 1) / share);
        }
    }
    const bool direct = a.direct && u0 == 0 && u1 == units;

    const int32_t* table = a.table + (a.whole ? 0 : (int64_t)set * a.max_blocks);
    u32x4 ks[STEPS], vs[STEPS];
    int entry = -1;
    uint32_t ok_next = 0;
    auto fetch_entry = [&](int i) {
        if (i < t1) entry = page_entry(a, table, a.dom_lo + tl.tile(i) * KT + (lane & 31), tl.khi);
    };
    auto stage = [&](int i) {
        const int j0 = a.dom_lo + tl.tile(i) * KT;
        const bool in = key_seen(a, tl, j0 + (lane & 31), pmin), good = in && (uint64_t)(int64_t)entry < (uint64_t)a.num_pages;
        if (a.err && in && !good) *a.err = 1;
        ok_next = (uint32_t)__ballot(good);
        load_tile<HD, SMALL, STEPS, 64>(a, j0, entry, ok_next, kvh, lane, ks, vs);
    };
    fetch_entry(t0 + wave);
    if (t0 + wave < t1) { stage(t0 + wave); fetch_entry(t0 + wave + 4); }

    u32x4 qf[NC][HD / 32];
    f32x4 o[NC][HD / 16];
    float m[NC], l[NC];
    #pragma unroll
    for (int n = 0; n < NC; ++n)
    {
        load_q<IO, HD, 32>(a, query_row(a, set, kvh, min(r0 + 16 * n + col, a.rows - 1)), quad, qf[n]);
        #pragma unroll
        for (int t = 0; t < HD / 16; ++t) o[n][t] = f32x4{};
        m[n] = -INFINITY;
        l[n] = 0.0f;
    }
    // K fragment: key row col (of 16), chunks 4 t + quad; V^T fragment: keys 4 quad + 0..3 (and + 16), columns 16 t + col
    const char* const krow = kl + col * RK + quad * 16;
    const char* const vrow = vl + (4 * quad + (col >> 2)) * RV + (col & 3) * 8;
    bool odd = false;
    for (int i = t0 + wave; i < t1; i += 4)
    {
        const uint32_t ok = ok_next;
        const int j = a.dom_lo + tl.tile(i) * KT;
        const bool whole = ok == 0xffffffffu && all_seen(a, j, KT, pmin, pmax);
        wave_lds_fence();
        if (!whole) odd |= clean_tile<IO, HD, STEPS, 64>(ks, vs, ok, lane);
        write_tile<HD, STEPS, 64, RV>(ks, vs, lane, kl, vl);
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
                const u32x4 kf = *(const u32x4*)(krow + k * 16 * RK + t * 64);
                #pragma unroll
                for (int n = 0; n < NC; ++n) s[n][k] = mfma16<IO>(kf, qf[n][t], s[n][k]);
            }
        }
        u32x4 pf[NC];
        #pragma unroll
        for (int n = 0; n < NC; ++n)
        {
            if (!whole)
            {
                const int p = pos[n], lo = a.window > 0 ? p - a.window + 1 : 0;
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
            mx = max_xor32(max_xor16(mx));
            if (__any(mx > m[n] + slack))
            {
                const float mn = fmaxf(m[n], mx), alpha = rescale_factor(m[n], mn, a.c);
                l[n] *= alpha;
                m[n] = mn;
                #pragma unroll
                for (int t = 0; t < HD / 16; ++t)
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][t][e] *= alpha;
            }
            const float base = exponent_base<IO>(m[n], a.c);
            float sum = 0.0f, pr[8];
            #pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                pr[e] = __builtin_amdgcn_exp2f(fmaf(s[n][e >> 2][e & 3], a.c, base));
                sum += pr[e];
            }
            l[n] += sum;
            #pragma unroll
            for (int e = 0; e < 4; ++e) pf[n][e] = pack2<IO>(pr[2 * e], pr[2 * e + 1]);
        }
        #pragma unroll
        for (int t = 0; t < HD / 16; ++t)
        {
            const auto v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr<s16x4>)(vrow + t * 32));
            const auto v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr<s16x4>)(vrow + 16 * RV + t * 32));
            const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
            const u32x4 vf = { w0.x, w0.y, w1.x, w1.y };
            #pragma unroll
            for (int n = 0; n < NC; ++n) o[n][t] = mfma16<IO>(vf, pf[n], o[n][t]);
        }
    }
    if (__any(odd))
        for (int i = t0 + wave; i < t1; i += 4)
            each_value_row<HD>(a, tl, table, a.dom_lo + tl.tile(i) * KT, KT, kvh, [&](int j, gcptr<uint16_t> v) {
                #pragma unroll
                for (int t = 0; t < HD / 16; ++t)
                    #pragma unroll
                    for (int e = 0; e < 4; ++e)
                    {
                        const uint16_t h = v[16 * t + 4 * quad + e];
                        if (!nonfinite<IO>(h)) continue;
                        #pragma unroll
                        for (int n = 0; n < NC; ++n)
                            if (row_sees(a, pos[n], j)) o[n][t][e] += load_bits<IO>(h);
                    }
            });
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
        // (kept above 0: an infinity of o stays one)
        const float f = fmaxf(__builtin_amdgcn_exp2f(fmaf(m[n], a.c, -ref)), 0x1p-126f);
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
    asm volatile("" : "+v"(tid));
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
        const QRow qr = query_row(a, set, kvh, r0 + r);
        const int64_t gr = qr.tok * a.hq + qr.h;
        if (direct)
        {
            const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
            if (a.lse && ch == 0) a.lse[gr] = ls == 0.0f ? -INFINITY : (rf - kShift<IO> + __builtin_amdgcn_logf(ls)) * kLn2;
            store_out4<IO>(a, qr.tok, qr.h, 4 * ch, sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
        }
        else
        {
            const int64_t pr = ((int64_t)kvh * (a.parts.slots + segs) + slot + g) * a.parts.seg_rows + r;
            if (ch == 0) { a.parts.ml[2 * pr] = fmaf(mm, a.c, -kShift<IO>); a.parts.ml[2 * pr + 1] = ls; }
            if (ls != 0.0f) ((gptr<f32x4>)(a.parts.po + pr * HD))[ch] = sum;
        }
    }
    start += units;
    if (start >= x1) break;
    __syncthreads();        // the next segment's tiles overwrite what was joined
    }
}

// ---------------------------------------------------------------------------------------------
// Joins the partial results of a row: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.  WAVES waves per row; a wave
// takes 256 / HD partial rows at a time (HD / 4 lanes of four columns each).  Measured: 4096 rows of 17 to 24 partial rows
// of 128 columns 9 us, 24528 rows of two of 256 columns 14 us (4.5 TB/s): bound by reading them.
struct JoinArgs
{
    Parts p[2];       // of the shared prefix (n 0 and no info: none), of the own keys
};

// A row's partial results of one launch: the first one's index, how many, the step between them.
struct PartList
{
    int64_t at, step;
    int n;
};

__device__ __forceinline__ PartList part_list(const AttnArgs& a, const Parts& p, int64_t gr, int b, int t, int h)
{
    PartList l{ gr * p.n, 1, p.n };
    if (p.info)
    {
        const int kvh = h / a.group, r = (p.whole ? b * a.seq + t : t) * a.group + (h - kvh * a.group), tile = r / p.seg_rows;
        const int seg = (p.whole ? 0 : b * p.row_tiles) + tile;
        const int first = p.info[2 * seg], last = p.info[2 * seg + 1];
        l.at = ((int64_t)kvh * (p.slots + p.segs) + first + seg) * p.seg_rows + (r - tile * p.seg_rows);
        l.step = p.seg_rows;
        l.n = last - first + 1;
    }
    return l;
}

template <class IO, int HD, int WAVES>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a, JoinArgs j)
{
    constexpr int LPR = HD / 4, SPW = 64 / LPR;       // lanes per partial row, partial rows per wave
    __shared__ float wt[4 / WAVES][2 * kMaxSplits];
    __shared__ f32x4 part[4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), local = wave / WAVES, sub = wave % WAVES;
    const int64_t gr = min((int64_t)blockIdx.x * (4 / WAVES) + local, a.rows_all - 1);
    const int tok = (int)(gr / a.hq), h = (int)(gr - (int64_t)tok * a.hq), b = tok / a.seq;
    const PartList pre = part_list(a, j.p[0], gr, b, tok - b * a.seq, h), own = part_list(a, j.p[1], gr, b, tok - b * a.seq, h);
    const int n0 = __builtin_amdgcn_readfirstlane(pre.n), ns = n0 + __builtin_amdgcn_readfirstlane(own.n);
    // A row that one slot had whole is written already.
    const bool done = a.direct && j.p[1].info && ns == 1;
    float m = -INFINITY, l = 0.0f;
    const auto ml = [&](int i) {
        return i < n0 ? ((gcptr<f32x2>)j.p[0].ml)[pre.at + i * pre.step] : ((gcptr<f32x2>)j.p[1].ml)[own.at + (i - n0) * own.step];
    };
    if (!done)
        for (int i = lane; i < ns; i += 64)
        {
            const f32x2 e = ml(i);
            if (e.y != 0.0f) m = fmaxf(m, e.x);
        }
    m = max_wave(m);
    if (!done)
        for (int i = lane; i < ns; i += 64)
        {
            const f32x2 e = ml(i);
            const float w = fmaxf(__builtin_amdgcn_exp2f(e.x - (m == -INFINITY ? 0.0f : m)), 0x1p-126f);   // as f above
            if (sub == 0) wt[local][i] = e.y != 0.0f ? w : -1.0f;      // -1: nothing was written
            if (e.y != 0.0f) l = fmaf(w, e.y, l);
        }
    l = group_sum<64>(l);
    __syncthreads();
    f32x4 o{};
    if (!done)
    {
        const gcptr<f32x4> p0 = (gcptr<f32x4>)(j.p[0].po + pre.at * HD) + lane % LPR, p1 = (gcptr<f32x4>)(j.p[1].po + own.at * HD) + lane % LPR;
        #pragma unroll 4
        for (int i = sub * SPW + lane / LPR; i < ns; i += WAVES * SPW)
        {
            const float w = wt[local][i];
            if (w < 0.0f) continue;
            const f32x4 p = i < n0 ? p0[i * pre.step * LPR] : p1[(i - n0) * own.step * LPR];
            #pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(w, p[e], o[e]);
        }
    }
    part[wave][lane] = o;
    __syncthreads();
    if (done || sub != 0 || lane >= LPR || (int64_t)blockIdx.x * (4 / WAVES) + local >= a.rows_all) return;
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
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (a.lse && lane == 0) a.lse[gr] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
    store_out4<IO>(a, tok, h, 4 * lane, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

}  // namespace exl3r

using namespace exl3r;

namespace {

struct Phase
{
    int cols;               // 0: k_attn_rows; 1, 2: k_attn_keys with that many column tiles
    int64_t sets, rows;     // row sets of `rows` query rows per KV head
    int64_t row_tiles;      // of a row set
    int64_t n;              // k_attn_rows: splits; k_attn_keys: slots per KV head
    bool cut;               // a row's keys may lie in several workgroups
    int64_t partials;       // partial rows in the workspace
    int64_t grid;
};

// How a phase is cut: `sets` row sets of `rows` query rows per KV head against at most `span` keys.
Phase plan_phase(int64_t sets, int64_t rows, int hk, int hd, int64_t span, bool whole)
{
    Phase p{};
    // (two column tiles of 256 dimensions do not fit the registers: two row tiles then, whose keys meet in the L2)
    p.cols = rows > 32 ? 0 : rows <= 16 || hd == 256 ? 1 : 2;
    p.sets = sets;
    p.rows = rows;
    if (p.cols == 0)
    {
        const int64_t tile = hd == 256 ? 128 : 256;
        p.row_tiles = (rows + tile - 1) / tile;
        const int64_t base = sets * hk * p.row_tiles, most = (span + 255) / 256;
        // A workgroup fills a CU.  The prefix's are equally long: no more than one round of them (16 x 37 tokens of 16
        // heads on a prefix of 2048: 6 splits 45 us, 7 splits, 280 workgroups, 55).  Others differ: at least one round.
        const int64_t fill = whole ? 256 / base : (256 + base - 1) / base;
        p.n = std::max<int64_t>(1, std::min<int64_t>({ fill, most, kMaxSplits }));
        p.cut = p.n > 1;
        p.partials = p.n * sets * rows * hk;
        p.grid = base * p.n;
    }
    else
    {
        const int64_t tile = 16 * p.cols;
        p.row_tiles = (rows + tile - 1) / tile;
        const int64_t segs = sets * p.row_tiles, units = (span + 127) / 128;
        // Two workgroups to a CU, as many as are resident; with more segments than that one each, as a slot starts its
        // segments one after the other.  (64 sequences of 700 to 8100 keys: 512 workgroups 221 us, 1024 225, 2048 232;
        // 2 sequences of 98765 and 131000: 100, 107, 123.)
        const int64_t want = std::max<int64_t>(512, std::min<int64_t>(segs * hk, 4096));
        p.n = std::max<int64_t>(1, std::min<int64_t>({ want / hk, segs * units, kMaxSplits }));
        p.cut = p.n > 1 && units > 1;
        p.partials = (p.n + segs) * hk * std::min(tile, rows);
        p.grid = p.n * hk;
    }
    return p;
}

struct Plan
{
    Phase prefix, own;      // prefix.n 0: none
    bool join;
    size_t bytes;
};

size_t phase_bytes(const Phase& p, int hd)
{
    const size_t info = p.cols ? ((size_t)p.sets * p.row_tiles * 8 + 255) & ~(size_t)255 : 0;
    return info + (((size_t)p.partials * (size_t)(hd + 2) * 4 + 255) & ~(size_t)255);
}

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
    p.own = plan_phase(bsz, seq * group, hk, hd, span, false);
    if (shared > 0) p.prefix = plan_phase(1, bsz * seq * group, hk, hd, shared, true);
    p.join = shared > 0 || p.own.cut;
    if (p.join) p.bytes = phase_bytes(p.own, hd) + (shared > 0 ? phase_bytes(p.prefix, hd) : 0);
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
    if (!(scale > 0.0f) || scale > 2.0e38f)     // (scale log2 e is finite too)
        return set_error(EXL3R_EINVAL, "%s: scale must be positive and finite", op);
    if (sinks < 0 || (window <= 0 && sinks != 0))
        return set_error(EXL3R_EINVAL, "%s: sinks (%d) must be 0 or more, and 0 without a window", op, sinks);
    if (hk > (1 << 22) / hd)        // (64 of a cache's rows are indexed in 32 bits)
        return set_error(EXL3R_EINVAL, "%s: KV heads of more than 2^22 elements together", op);
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
    // (2^23: a launch has fewer than 2^32 threads, 512 in a workgroup)
    if (p.own.grid > 0x7fffff || p.prefix.grid > 0x7fffff || (p.join && tokens * hq > 0xffffff))
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
    a.q_ts = q_ts; a.q_hs = q_hs; a.o_ts = o_ts; a.o_hs = o_hs;
    a.max_blocks = max_blocks;
    a.num_pages = num_pages;
    a.bsz = (int)bsz; a.seq = (int)seq; a.hq = hq; a.hk = hk; a.group = (int)group;
    a.page_shift = __builtin_ctz((unsigned)page_size);
    a.window = window > 0 ? window : 0;
    a.sinks = sinks;
    a.direct = shared == 0;
    a.q_vec = aligned16(q) && (hq == 1 || q_hs % 8 == 0) && (tokens == 1 || q_ts % 8 == 0);
    a.o_vec = ((uintptr_t)out & 7) == 0 && (hq == 1 || o_hs % 4 == 0) && (tokens == 1 || o_ts % 4 == 0);
    a.c = scale * 1.4426950408889634f;
    hipStream_t st = (hipStream_t)stream;

    auto run = [&](auto T, auto HDC) {
        using IO = decltype(T);
        constexpr int HD = decltype(HDC)::value;
        char* place = (char*)ws;
        auto phase = [&](const Phase& ph, bool whole, int64_t lo, int64_t hi) {
            AttnArgs x = a;
            x.whole = whole;
            x.dom_lo = (int)lo;
            x.dom_hi = (int)hi;
            x.rows = (int)ph.rows;
            x.row_tiles = (int)ph.row_tiles;
            Parts& pt = x.parts;
            const int64_t segs = ph.sets * ph.row_tiles;
            if (ph.cols)
            {
                pt.slots = (int)ph.n;
                pt.segs = (int)segs;
                pt.row_tiles = (int)ph.row_tiles;
                pt.seg_rows = (int)std::min<int64_t>(16 * ph.cols, ph.rows);
                pt.whole = whole;
            }
            else
            {
                pt.n = (int)ph.n;
                x.direct = !p.join;
            }
            if (p.join)
            {
                char* at = place;
                if (ph.cols)
                {
                    pt.info = (int32_t*)at;
                    at += (segs * 8 + 255) & ~(int64_t)255;
                }
                pt.po = (float*)at;
                pt.ml = pt.po + ph.partials * hd;
                place += phase_bytes(ph, hd);
            }
            const int64_t grid = ph.grid;
            if (ph.cols == 0)
            {
                constexpr int W = HD == 256 ? 4 : 8, KT = HD == 256 ? 32 : 64;
                if (page_size < KT) launch(k_attn_rows<IO, HD, W, KT, true>, (unsigned)grid, 64 * W, 0, st, x);
                else launch(k_attn_rows<IO, HD, W, KT, false>, (unsigned)grid, 64 * W, 0, st, x);
            }
            else if (ph.cols == 1)
            {
                if (page_size < 32) launch(k_attn_keys<IO, HD, 1, true>, (unsigned)grid, 256, 0, st, x);
                else launch(k_attn_keys<IO, HD, 1, false>, (unsigned)grid, 256, 0, st, x);
            }
            else if constexpr (HD != 256)
            {
                if (page_size < 32) launch(k_attn_keys<IO, HD, 2, true>, (unsigned)grid, 256, 0, st, x);
                else launch(k_attn_keys<IO, HD, 2, false>, (unsigned)grid, 256, 0, st, x);
            }
            return pt;
        };
        JoinArgs j{};
        if (shared > 0) j.p[0] = phase(p.prefix, true, 0, shared);
        j.p[1] = phase(p.own, false, shared, cap);
        if (p.join)
        {
            // Many partial results of few rows: 4 waves each.  (16 + up to 8 of 4096 rows: 12 us so, 9 with one wave.)
            if (p.own.n + p.prefix.n > 16 && a.rows_all <= 1024) launch(k_attn_join<IO, HD, 4>, (unsigned)a.rows_all, 256, 0, st, a, j);
            else launch(k_attn_join<IO, HD, 1>, (unsigned)((a.rows_all + 3) / 4), 256, 0, st, a, j);
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
