// Attention of a tree of drafted tokens over the KV cache.
//
// Row (b, t, h): s_j = q . k_j / sqrt(hd) over the visible positions j, p_j = exp(s_j - max s),
// out = sum p_j v_j / sum p_j; a row that sees nothing is zero.
//
// All rows of a sequence that share a kv head share its K / V stream, so the work is cut into
// units (sequence, kv head, row tile) and each unit into tiles of positions.  The tiles of all
// units, in order, are dealt out to the CTAs in equal contiguous ranges: lengths are read on the
// device, ragged batches stay balanced, and a range that begins or ends inside a unit leaves a
// partial result (row maximum, sum, weighted V) for tf_tree_combine_kernel, in a fixed order.
//
// Arithmetic (fp32-equivalent on the f16 tensor pipe): an operand is split into two f16 halves
// after a power-of-two scale (q: per row; fp32 K and V: per tile; p: fixed), 22 bits or more of
// it; the product of the two low halves (2^-22 relative) is dropped.  An f16 cache is its own
// exact half; a bf16 row fits one half after the scale (8 bits; f16 runs out of exponents 2^-24
// below 1).  Every tile's P V product starts from zero and joins the running output by an fp32
// fma, so its rounding does not grow with the context.
// One scale serves a tile whose rows' maxima lie within 2^12 of each other.  Beyond that the small
// rows would lose their bits to a large one, which need not have a reader in common with them: a
// segment with such a tile is computed once more from the cache, in fp32 and row by row
// (tree_exact_rows).  A probability below 2^-39 of its row's largest counts as zero.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <cstring>

#include "tree.cuh"

namespace tfb {

constexpr int TN_THREADS = 256;
// Tiles that a unit's start and end (queries, partial results, output) take the time of in the narrow
// and the wide kernel.  Without them / with them, device time: 1 tree of 8, 8000 positions, 32x8x64 f32
// (narrow) 28.7 / 22.9 us; 12 trees of 31, 4001 positions, 32x8x128 bf16 (wide) 113 / 97 us; 32 trees
// of 64, 8128 positions, 32x8x64 f16 (wide) 257 / 212 us; 1 tree of 64, 16000 positions 48.8 / 50.7 us.
constexpr int TN_UNIT_COST = 2;
constexpr int TW_UNIT_COST = 5;
constexpr int TN_TILE_BYTES = 32768;  // K and V bytes of a tile in the cache's type: 32 registers per thread
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 15.f;       // p is held as 2^15 exp(s - max): its low half keeps 2^-24 / 2^15 of it

// ---- the split of the tiles over the CTAs ---------------------------------------------------------
struct TreePlan {
    int maps;                // wide kernel, 16-bit cache: the tensor maps are valid
    int slot_rows;           // rows of the tensor maps per slot
    int grid;                // CTAs of the main kernel
    int rt;                  // rows per row tile
    int rep;                 // query heads per kv head
    int rep_inv;             // (x * rep_inv) >> 16 = x / rep for x < 2048 and rep <= 8
};
struct TreeDesc {            // a unit split over CTAs c0..c1, found at slot c0
    int b, kvh, tile, c1;    // b < 0: none; tile: row tile, and its rows in the high half
};

__host__ __device__ inline size_t tree_part_floats(int rt, int hd) { return (size_t)rt * (hd + 2); }

struct TreeSeq {
    int slot, n_ctx, n_node;  // n_node 0: nothing to do (or a bad sequence)
    bool bad;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeAttnArgs& a, int b) {
    TreeSeq s;
    s.slot = a.slots ? a.slots[b] : b;
    s.n_ctx = a.n_ctx[b];
    s.n_node = a.n_node ? min(a.n_node[b], a.T) : a.T;
    s.bad = s.slot < 0 || s.slot >= a.n_slots || s.n_ctx < 0 || s.n_node < 0 || s.n_ctx > a.cap - s.n_node;
    if (s.bad) s.n_node = 0;
    return s;
}
// tiles of one unit of the sequence, and its units
template <int PT>
__device__ __forceinline__ int seq_tiles(const TreeSeq& s) {
    return s.n_node ? (unsigned)(s.n_ctx + s.n_node + PT - 1) / PT : 0;
}
template <int RT>
__device__ __forceinline__ int seq_units(int n_kv, int rep, const TreeSeq& s) {
    return n_kv * ((unsigned)(s.n_node * rep + RT - 1) / RT);
}

// A CTA's place in its range of tiles [g0, g1): the sequence it is in and the global index of
// that sequence's first tile.  (32 bits: tree_attn_fits.)
struct TreeIter {
    int g0, g1, per, base, b;
};
// The next piece of the range: tiles [t0, t1) of one unit.
struct TreeSeg {
    TreeSeq s;
    int b, kvh, rtile, t0, t1, tiles, last_cta;  // last_cta: the CTA that ends the unit
};

// Each unit counts for its tiles and UC more, the time (in tiles) that starting and ending a unit
// takes.  Finds this CTA's range; every warp by itself, lanes over the sequences.
template <int PT, int RT, int UC>
__device__ __forceinline__ void tree_range(const TreeAttnArgs& a, const TreePlan& pl, TreeIter& it) {
    const int lane = threadIdx.x & 31;
    const int chunk = (a.B + 31) >> 5, lo = min(a.B, lane * chunk), hi = min(a.B, lo + chunk);
    int mine = 0, units = 0;
#pragma unroll 1
    for (int b = lo; b < hi; ++b) {
        const TreeSeq s = tree_seq(a, b);
        if (s.n_node) {
            const int u = seq_units<RT>(a.n_kv, pl.rep, s);
            mine += (seq_tiles<PT>(s) + UC) * u;
            units += u;
        }
        if (s.bad && blockIdx.x == 0 && threadIdx.x < 32) atomicCAS(a.err, 0, ERR_POS);
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
    }
    const int total = __shfl_sync(0xFFFFFFFFu, inc, 31);
    // (units of two tiles and less stay whole: a split unit costs the second kernel's work)
    units = __reduce_add_sync(0xFFFFFFFFu, units);
    const int least = total - units * UC <= 2 * units ? 2 + UC : 2;
    it.per = max((int)((unsigned)(total + pl.grid - 1) / (unsigned)pl.grid), least);
    it.g0 = (int)min((long long)it.per * blockIdx.x, (long long)total);
    it.g1 = min(it.g0 + it.per, total);
    // the lane whose sequences hold g0, then the sequence
    const unsigned in = __ballot_sync(0xFFFFFFFFu, it.g0 < inc);
    const int src = in ? __ffs(in) - 1 : 31;
    int base = inc - mine, b = lo;
    if (lane == src)
#pragma unroll 1
        for (; b + 1 < hi; ++b) {
            const TreeSeq s = tree_seq(a, b);
            const int t = s.n_node ? (seq_tiles<PT>(s) + UC) * seq_units<RT>(a.n_kv, pl.rep, s) : 0;
            if (it.g0 < base + t) break;
            base += t;
        }
    it.b = __shfl_sync(0xFFFFFFFFu, b, src);
    it.base = __shfl_sync(0xFFFFFFFFu, base, src);
}

template <int PT, int RT, int UC>
__device__ __forceinline__ bool tree_next(const TreeAttnArgs& a, int rep, TreeIter& it, TreeSeg& o) {
#pragma unroll 1
    while (it.g0 < it.g1) {
        o.s = tree_seq(a, it.b);
        o.tiles = seq_tiles<PT>(o.s);
        const int nrt = (unsigned)(o.s.n_node * rep + RT - 1) / RT, cost = o.tiles + UC;
        if (!o.s.n_node || it.g0 >= it.base + cost * a.n_kv * nrt) {  // next sequence
            if (o.s.n_node) it.base += cost * a.n_kv * nrt;
            ++it.b;
            continue;
        }
        const int unit = (unsigned)(it.g0 - it.base) / (unsigned)cost;
        const int u0 = it.base + unit * cost;  // the unit's start
        o.t0 = max(0, it.g0 - u0 - UC);
        o.t1 = min(it.g1 - u0, cost) - UC;
        it.g0 = min(it.g1, u0 + cost);
        if (o.t1 <= o.t0) continue;
        o.b = it.b;
        o.kvh = (unsigned)unit / (unsigned)nrt;
        o.rtile = unit - o.kvh * nrt;
        o.last_cta = (unsigned)(u0 + cost - 1) / (unsigned)it.per;
        return true;
    }
    return false;
}

// Rows that no unit covers (nodes from n_node on, bad sequences) are zero.
template <int NT>
__device__ __forceinline__ void tree_zero_rows(const TreeAttnArgs& a) {
    const int n4 = a.n_head * a.hd / 4, per = NT / 32;
#pragma unroll 1
    for (long long r = (long long)blockIdx.x * per + (threadIdx.x >> 5); r < (long long)a.B * a.T; r += (long long)gridDim.x * per) {
        const TreeSeq s = tree_seq(a, (int)(r / a.T));
        if ((int)(r % a.T) < s.n_node) continue;
        float4* o = reinterpret_cast<float4*>(a.out + r * a.ld_out);
#pragma unroll 1
        for (int i = threadIdx.x & 31; i < n4; i += 32) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
}

// What a row sees of the drafted nodes, as 32-bit words in shared memory: words 1 .. 8 hold nodes
// 0 .. 255 (none from n_node on), word 0 all ones for the committed positions before them, word 9
// zero for what lies behind.
constexpr int VIS_WORDS = TREE_MAX_NODES / 32 + 2;
__device__ __forceinline__ void vis_fill(uint32_t* vis, const TreeAttnArgs& a, const TreeSeq& s, int b, int node) {
    vis[0] = 0xFFFFFFFFu;
    vis[VIS_WORDS - 1] = 0;
    const uint32_t* mw = a.mask ? reinterpret_cast<const uint32_t*>(a.mask + ((size_t)b * a.T + node) * ((a.T + 63) / 64)) : nullptr;
#pragma unroll 1
    for (int w = 0; w < TREE_MAX_NODES / 32; ++w) {
        uint32_t v = 0;
        const int left = s.n_node - 32 * w;
        if (left > 0 && node < s.n_node) {
            if (mw) v = mw[w];
            else v = node < 32 * w ? 0u : (node - 32 * w >= 31 ? 0xFFFFFFFFu : (2u << (node - 32 * w)) - 1);
            if (left < 32) v &= (1u << left) - 1;
        }
        vis[w + 1] = v;
    }
}
// the 32 positions from drafted index x0 on (negative: committed)
__device__ __forceinline__ uint32_t vis_window(const uint32_t* vis, int x0) {
    if (x0 <= -32) return 0xFFFFFFFFu;
    const int w = min((x0 >> 5) + 1, VIS_WORDS - 2);
    return x0 >= TREE_MAX_NODES ? 0u : __funnelshift_r(vis[w], vis[w + 1], x0 & 31);
}

// Bounded wait on an mbarrier phase with the hardware's own suspension (up to 20 us a try, 2^16
// tries); false after a timeout, or when another thread of the block gave up.
__device__ __forceinline__ bool tree_wait(uint64_t* bar, int parity, int* err, int code, volatile int* abort) {
#pragma unroll 1
    for (int i = 0; i < 65536; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity & 1)
            : "memory");
        if (ok) return true;
        if (abort && *abort) return false;
    }
    atomicCAS(err, 0, code);
    if (abort) *abort = 1;
    return false;
}

// Takes the non-finite values of drafted rows, which the operands hold as zeros, up in the rows
// that see them: adds them to what has been written of the segment's rows (after a barrier).
template <int KVT>
__device__ __forceinline__ void tree_fix_rows(const TreeAttnArgs& a, const TreeSeg& sg, int rt, int rep, const unsigned* badrow,
                                           const uint32_t* vis, float* part, bool whole, int tid, int threads) {
    const int hd = a.hd, rows = sg.s.n_node * rep;
#pragma unroll 1
    for (int i = tid; i < rt * hd; i += threads) {
        const int r = i / hd, d = i - r * hd, rr = sg.rtile * rt + r, node = rr / rep;
        if (rr >= rows) return;
        float* dst = whole ? a.out + ((size_t)sg.b * a.T + node) * a.ld_out + (size_t)(sg.kvh * rep + rr - node * rep) * hd + d : part + i;
#pragma unroll 1
        for (int w = 0; w < TREE_MAX_NODES / 32; ++w)
#pragma unroll 1
            for (unsigned bits = badrow[w] & vis[r * VIS_WORDS + w + 1]; bits; bits &= bits - 1) {
                const float v = kv_load(a.vc, (long long)sg.s.slot * a.slot_stride +
                                                  ((long long)sg.kvh * a.cap + sg.s.n_ctx + 32 * w + __ffs(bits) - 1) * hd + d, KVT);
                if (!(fabsf(v) < INFINITY)) *dst += v;
            }
    }
}

// ---- small pieces ---------------------------------------------------------------------------------
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e for -126 <= e <= 127
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
// Whether a tile whose largest |x| is maxbits may be split after the scale 2^-e: its maximum within
// [2^8, 2^15), so that nothing overflows and the low halves keep 20 bits of every row whose own
// maximum is at most 2^TILE_SPREAD below it; and an exponent that puts it in the middle.
constexpr int TILE_SPREAD = 12;
constexpr int TILE_FIRST = -9;  // the exponent before the first tile
__device__ __forceinline__ bool tile_fits(uint32_t maxbits, int e) {
    const int x = (int)(maxbits >> 23) - 127 - e;
    return maxbits == 0 || (x < 15 && (x >= 8 || e == -126));
}
__device__ __forceinline__ int tile_exponent(uint32_t maxbits) {
    const int e = (int)(maxbits >> 23) - 127 - 11;
    return e < -126 ? -126 : (e > 126 ? 126 : e);
}
// Whether a vector whose largest |x| is `bits` leaves open that its row keeps fewer bits.
__device__ __forceinline__ bool may_be_low(uint32_t bits, int e) { return (int)(bits >> 23) - 127 < e + 8 - TILE_SPREAD; }
// exponent e such that |x| 2^-e lies in [2^14, 2^15) for the largest finite |x| (its bits
// without sign), kept where 2^e and 2^-e are normal numbers
__device__ __forceinline__ int half_exponent(uint32_t maxbits) {
    const int e = (int)(maxbits >> 23) - 127 - 14;
    return e < -126 ? -126 : (e > 126 ? 126 : e);
}
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
    return b >= 0x7F800000u ? 0u : b;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Two values in halves: the high one by truncation, 10 bits behind the first (exact in f16 from
// 2^-14 on), the low one the rest.
__device__ __forceinline__ void split2t(float2 x, uint32_t& hi, uint32_t& lo) {
    const float2 h = make_float2(__uint_as_float(__float_as_uint(x.x) & 0xFFFFE000u), __uint_as_float(__float_as_uint(x.y) & 0xFFFFE000u));
    const float2 l = __fadd2_rn(x, make_float2(-h.x, -h.y));
    hi = pack_half2(h.x, h.y);
    lo = pack_half2(l.x, l.y);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in) {  // zeros when !in
    const int n = in ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, const uint32_t (&w)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t src) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
    return v;
}
// Zeroes the non-finite values of a vector of type KVT; whether there were any.
template <int KVT>
__device__ __forceinline__ bool zero_nonfinite(uint4& x) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&x);
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (KVT == KV_F32) {
            if ((w[j] & 0x7F800000u) == 0x7F800000u) bad = true, w[j] = 0;
        } else {
            const uint32_t em = KVT == KV_F16 ? 0x7C00u : 0x7F80u;
            if ((w[j] & em) == em) bad = true, w[j] &= 0xFFFF0000u;
            if ((w[j] >> 16 & em) == em) bad = true, w[j] &= 0xFFFFu;
        }
    }
    return bad;
}
// largest finite |x| of a vector of type KVT (fp32 or bf16), as fp32 bits
template <int KVT>
__device__ __forceinline__ uint32_t max_bits(const uint4& x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (KVT == KV_F32) m = max(m, finite_abs_bits(__uint_as_float(w[j])));
        else m = max(m, max(finite_abs_bits(__uint_as_float(w[j] << 16)), finite_abs_bits(__uint_as_float(w[j] & 0xFFFF0000u))));
    }
    return m;
}
// |x| of a vector's largest value, as fp32 bits (fp32 or bf16; 0x7F800000 and more: not all finite;
// fp32: NaN aside where there is another value)
template <int KVT>
__device__ __forceinline__ uint32_t abs_bits(const uint4& x) {
    if (KVT == KV_F32)
        return __float_as_uint(fmaxf(fmaxf(fabsf(__uint_as_float(x.x)), fabsf(__uint_as_float(x.y))),
                                     fmaxf(fabsf(__uint_as_float(x.z)), fabsf(__uint_as_float(x.w)))));
    const uint32_t m = 0x7FFF7FFFu;
    const uint32_t v = __vmaxu2(__vmaxu2(x.x & m, x.y & m), __vmaxu2(x.z & m, x.w & m));
    return max(v << 16, v & 0xFFFF0000u);
}
// running maximum of |x| over vectors, cheaper: fp32 as a float, bf16 as two packed values whose
// signs are not meaningful; NaN aside
template <int KVT>
__device__ __forceinline__ void abs_max(uint32_t& m, const uint4& x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (KVT == KV_F32) m = __float_as_uint(fmaxf(__uint_as_float(m), fabsf(__uint_as_float(w[j]))));
        else asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w[j]));
    }
}
template <int KVT>
__device__ __forceinline__ uint32_t abs_max_bits(uint32_t m) {
    return KVT == KV_F32 ? m : max((m << 16) & 0x7FFF0000u, m & 0x7FFF0000u);
}
// largest |x| of eight values (NaN aside), as fp32 bits
__device__ __forceinline__ uint32_t max8(const float4& x, const float4& y) {
    return __float_as_uint(fmaxf(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))),
                                 fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)))));
}
// eight values times f in two halves
__device__ __forceinline__ void split8(const float4& x, const float4& y, float f, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    const float2 g = make_float2(f, f);
    split2t(__fmul2_rn(make_float2(x.x, x.y), g), hi[0], lo[0]);
    split2t(__fmul2_rn(make_float2(x.z, x.w), g), hi[1], lo[1]);
    split2t(__fmul2_rn(make_float2(y.x, y.y), g), hi[2], lo[2]);
    split2t(__fmul2_rn(make_float2(y.z, y.w), g), hi[3], lo[3]);
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// four consecutive elements of the cache
template <int KVT>
__device__ __forceinline__ float4 kv_load4(const void* p, long long i) {
    if (KVT == KV_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u));
}
// Whether a tile of the segment has rows whose maxima lie further apart than its scale allows (rows of
// zeros aside): a warp's share of the tiles, a lane per row.  (The look at one vector of a row finds
// channels of small values too: with 16 of 64 at 10^-9 a call of 1 tree of 64, 16000 positions takes
// 91 us instead of 58.)
template <int KVT, int PT>
__device__ __noinline__ bool tree_rows_apart(const TreeAttnArgs& a, const TreeSeg sg, int warp, int warps) {
    const int hd = a.hd, end = sg.s.n_ctx + sg.s.n_node, lane = threadIdx.x & 31;
    const long long base = (long long)sg.s.slot * a.slot_stride + (long long)sg.kvh * a.cap * hd;
    bool apart = false;
#pragma unroll 1
    for (int i = 2 * sg.t0 + warp; i < 2 * sg.t1; i += warps) {  // tile, K / V
        const void* c = i & 1 ? a.vc : a.kc;
        uint32_t hi = 0, lo = 0xFFFFFFFFu;
#pragma unroll 1
        for (int p = (i >> 1) * PT + lane; p < min(((i >> 1) + 1) * PT, end); p += 32) {
            uint32_t m = 0;
#pragma unroll 4
            for (int d = 0; d < hd; d += 4) {
                const float4 x = kv_load4<KVT>(c, base + (long long)p * hd + d);
                m = max(m, max(max(finite_abs_bits(x.x), finite_abs_bits(x.y)), max(finite_abs_bits(x.z), finite_abs_bits(x.w))));
            }
            hi = max(hi, m);
            if (m) lo = min(lo, m);
        }
        hi = __reduce_max_sync(0xFFFFFFFFu, hi);
        lo = __reduce_min_sync(0xFFFFFFFFu, lo);
        apart |= hi && (int)(hi >> 23) - (int)(lo >> 23) > TILE_SPREAD;
    }
    return apart;
}
// A segment's rows in fp32, over what has been written of them (after a barrier): for tiles whose rows
// lie too far apart for one scale.  Four rows per warp, which share the cache's loads; 32 positions
// at a time, a lane per position for the scores and per dim (d, d + 32, ...) for the sums.  (fp32
// and bf16 caches.)  Bound by the latency of its loads; calls without / with one row 10^6 times the
// others: 1 tree of 8, 8000 positions, 32x8x64 f32 30 / 119 us; 32 trees of 8, 1144 positions,
// 12x2x128 f32 54 / 500 us; 1 tree of 64, 16000 positions, 32x8x64 f32 58 / 2150 us; 12 trees of 31,
// 4001 positions, 32x8x128 bf16 122 / 7000 us.  A function of its own, so that the kernels' loops keep
// their registers.
template <int KVT, int PT>
__device__ __noinline__ void tree_exact_rows(const TreeAttnArgs& a, const TreeSeg sg, int rt, int rep, const uint32_t* vis, float* part,
                                                bool whole, int warp, int warps) {
    constexpr int R = 4;
    const int hd = a.hd, rows = min(rt, sg.s.n_node * rep - sg.rtile * rt), lane = threadIdx.x & 31;
    const int p1 = min(sg.t1 * PT, sg.s.n_ctx + sg.s.n_node);
    const long long base = (long long)sg.s.slot * a.slot_stride + (long long)sg.kvh * a.cap * hd;
    const float scale = kLog2e / sqrtf((float)hd);
#pragma unroll 1
    for (int r0 = warp * R; r0 < rows; r0 += warps * R) {
        const float* q[R];
        float m[R], l[R], o[R][4];
#pragma unroll
        for (int i = 0; i < R; ++i) {  // (the last row stands in for rows behind it)
            const int rr = sg.rtile * rt + min(r0 + i, rows - 1), node = rr / rep;
            q[i] = a.q + ((size_t)sg.b * a.T + node) * a.ld_q + (size_t)(sg.kvh * rep + rr - node * rep) * hd;
            m[i] = -INFINITY;
            l[i] = o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        }
#pragma unroll 1
        for (int p0 = sg.t0 * PT; p0 < p1; p0 += 32) {
            const int p = min(p0 + lane, p1 - 1);
            float s[R] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int d = 0; d < hd; d += 4) {
                const float4 k = kv_load4<KVT>(a.kc, base + (long long)p * hd + d);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(q[i] + d);
                    s[i] = fmaf(x.x, k.x, fmaf(x.y, k.y, fmaf(x.z, k.z, fmaf(x.w, k.w, s[i]))));
                }
            }
            unsigned seen[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t bits = vis_window(vis + min(r0 + i, rows - 1) * VIS_WORDS, p0 - sg.s.n_ctx);
                seen[i] = p1 - p0 < 32 ? bits & ((1u << (p1 - p0)) - 1) : bits;
                const bool mine = seen[i] >> lane & 1;
                const float x = mine ? s[i] * scale : -INFINITY;
                const float mx = fmaxf(m[i], warp_max(x)), ref = mx == -INFINITY ? 0.f : mx, alpha = exp2_fast(m[i] - ref);
                s[i] = mine ? exp2_fast(x - ref + kPShift) : 0.f;  // the weight from here on
                m[i] = mx;
                l[i] = fmaf(l[i], alpha, warp_sum(s[i]));
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] *= alpha;
            }
#pragma unroll 4
            for (int j = 0; j < 32; ++j) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = lane + 32 * e < hd ? kv_load(a.vc, base + (long long)min(p0 + j, p1 - 1) * hd + lane + 32 * e, KVT) : 0.f;
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float w = __shfl_sync(0xFFFFFFFFu, s[i], j);
                    if (seen[i] >> j & 1)  // (what is not seen may not be finite)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][e] = fmaf(w, v[e], o[i][e]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = r0 + i, rr = sg.rtile * rt + r, node = rr / rep;
            if (r >= rows) continue;
            const float inv = !whole ? 1.f : (l[i] == 0.f ? 0.f : 1.f / l[i]);
            float* dst = whole ? a.out + ((size_t)sg.b * a.T + node) * a.ld_out + (size_t)(sg.kvh * rep + rr - node * rep) * hd : part + (size_t)r * hd;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (lane + 32 * e < hd) dst[lane + 32 * e] = o[i][e] * inv;
            if (!whole && lane == 0) {
                part[(size_t)rt * hd + r] = m[i];
                part[(size_t)rt * hd + rt + r] = l[i];
            }
        }
    }
}

// ---- narrow trees: mma.sync, up to 64 rows per row tile ----------------------------------------------
// (16 rows do not fill a tcgen05 product, and its set-up costs more than a short context takes.)
// One CTA of 8 warps per range of tiles, two CTAs per SM.  A tile is 32 KB of cache (K and V),
// copied into shared memory by cp.async one tile ahead while the current one is computed; fp32
// and bf16 tiles are then split into f16 halves in a second buffer, each thread taking the
// vectors that it copied itself (no barrier in between), f16 tiles alternate between the two
// buffers.  Operand rows are HD halves, 16-byte chunk c of row r at c ^ (r & 7).
// Warp (m, g): 16 rows of row block m, the positions of group g of the tile; each keeps its own
// running maximum, sum and output, and the groups meet through shared memory when a unit ends.
// 32 KB tiles, because two CTAs of two buffers and the queries fill an SM's shared memory.
//
// Bound by the latency of a tile's chain (copy, split, scores, softmax, P V: about 6000 cycles per
// tile and CTA, two CTAs per SM) and, in short calls, by the unit's start (queries behind the
// lengths, 5000 cycles) and the launches.  Device time, both launches: 1 tree of 1, 96 positions,
// 32x8x64 f32 8.8 us; 1 tree of 5, 1733 positions, 14x2x64 f32 13.3 us; 1 tree of 8, 8000 positions,
// 32x8x64 f32 23.3 us (33 MB: 1.4 TB/s); 32 ragged trees of 8, 1144 positions, the same 46.0 us (91
// MB: 2.0 TB/s).  The look at the range of a tile's rows (TILE_SPREAD) is 1 to 4 % of that.
template <int HD, int MT, int KVT>
struct NarrowCfg {
    static constexpr int ESZ = KVT == KV_F32 ? 4 : 2;
    static constexpr int PT = TN_TILE_BYTES / (2 * HD * ESZ);
    static constexpr int RT = 16 * MT;
    static constexpr int NG = (PT / 16) < (8 / MT) ? (PT / 16) : (8 / MT);  // position groups
    static constexpr int PW = PT / NG;                                     // positions per warp and tile
    static constexpr int PB = PW < 32 ? PW : 32;                           // per softmax step
    static constexpr int NLO = KVT == KV_F32 ? 2 : 1;                      // halves of a cache element
    static constexpr int TILE_H = PT * HD * 2;                             // bytes of one half of a tile
    static constexpr int Q_BYTES = RT * HD * 2;
    static constexpr int FIN = NG * RT * (HD + 4) * 4;
    static constexpr int MAIN = 2 * TN_TILE_BYTES + 2 * Q_BYTES;           // two tile buffers, q halves
    static constexpr int SMEM = MAIN > FIN ? MAIN : FIN;
};

template <int HD, int MT, int KVT>
__global__ void __launch_bounds__(TN_THREADS, 2)
    tf_tree_attn_narrow_kernel(const __grid_constant__ TreeAttnArgs a, const __grid_constant__ TreePlan pl) {
    using F = NarrowCfg<HD, MT, KVT>;
    constexpr int PT = F::PT, RT = F::RT, NG = F::NG, PB = F::PB, NLO = F::NLO, ESZ = F::ESZ;
    constexpr int VEC = 16 / ESZ, VPR = HD / VEC, NV = TN_TILE_BYTES / 2 / 16 / TN_THREADS;  // vectors: elements, per row, per thread
    constexpr uint32_t HALF_TILE = TN_TILE_BYTES / 2;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ float qscale[RT];
    __shared__ uint32_t vis[RT][VIS_WORDS];
    __shared__ unsigned tmax[4];                      // maxima of K, V (bits) of this tile and the next
    __shared__ int low;                               // the segment may have a tile whose rows one scale does not hold
    __shared__ unsigned badrow[TREE_MAX_NODES / 32];  // drafted rows of the unit with non-finite values
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rep = pl.rep, hd = a.hd;
    const uint32_t sb = smem_u32(smem);
    const uint32_t qh = sb + 2 * TN_TILE_BYTES, ql = qh + F::Q_BYTES;
    const int rep_inv = pl.rep_inv;
    auto div_rep = [&](int x) { return (x * rep_inv) >> 16; };
    const int wm = warp % MT, wg = warp / MT;  // row block, position group
    const int g8 = lane >> 2, q4 = lane & 3;

    pdl_trigger();
    pdl_wait();
    TreeDesc* desc = static_cast<TreeDesc*>(a.ws);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + 65536);
    TreeIter it;
    tree_range<PT, RT, TN_UNIT_COST>(a, pl, it);
    if (tid == 0) desc[blockIdx.x].b = -1;

    TreeSeg sg;
    int ek = KVT == KV_F16 ? 0 : TILE_FIRST, ev = ek;  // scale exponents of K and V, kept from tile to tile
    while (tree_next<PT, RT, TN_UNIT_COST>(a, rep, it, sg)) {
        const TreeSeq s = sg.s;
        const int b = sg.b, kvh = sg.kvh, rtile = sg.rtile, t0 = sg.t0, t1 = sg.t1;
        const int end = s.n_ctx + s.n_node, rows = s.n_node * rep;
        const bool active = wg < NG && rtile * RT + wm * 16 < rows;  // (a row block behind the last row is left out)
        const size_t off = (size_t)s.slot * a.slot_stride + (size_t)kvh * a.cap * hd;
        const uint8_t* kp = static_cast<const uint8_t*>(a.kc) + off * ESZ;
        const uint8_t* vp = static_cast<const uint8_t*>(a.vc) + off * ESZ;

        // tile t into its buffer: vector v = tid + i * threads of the PT x HD tile, K then V
        // (f16: at its operand place, the buffers alternating; else in the order of the threads)
        const int r0 = tid / VPR, c0 = tid % VPR;
        constexpr int RSTEP = TN_THREADS / VPR;  // a multiple of 8: chunk c0 stays at c0 ^ (r0 & 7)
        const uint32_t own = KVT == KV_F16 ? sb + (uint32_t)r0 * (HD * 2) + (uint32_t)((c0 ^ (r0 & 7)) << 4) : sb + 16u * tid;
        constexpr uint32_t OSTEP = KVT == KV_F16 ? RSTEP * HD * 2 : 16 * TN_THREADS;
        auto load = [&](int t) {
            const uint32_t o = own + (KVT == KV_F16 ? (uint32_t)(t & 1) * TN_TILE_BYTES : 0u);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int p = t * PT + r0 + i * RSTEP;
                const bool in = p < end && c0 * VEC < hd;
                const size_t e = in ? ((size_t)p * hd + c0 * VEC) * ESZ : 0;
                cp_async16(o + i * OSTEP, kp + e, in);
                cp_async16(o + i * OSTEP + HALF_TILE, vp + e, in);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        load(t0);
        // the rows' queries, TPR threads per row: scaled to [2^14, 2^15), two halves; what they see
        {
            constexpr int TPR = TN_THREADS / RT < HD / 8 ? TN_THREADS / RT : HD / 8, UPT = HD / 8 / TPR;  // 8-dim units per thread
            const int r = tid / TPR, rr = rtile * RT + r, j0 = tid % TPR;
            if (r < RT) {
                float4 x[UPT][2];
                uint32_t mb = 0;
                const int node = div_rep(rr);
                const float* qp = a.q + ((size_t)b * a.T + node) * a.ld_q + (size_t)(kvh * rep + rr - node * rep) * hd;
#pragma unroll
                for (int i = 0; i < UPT; ++i) {
                    const int d = (j0 + i * TPR) * 8;
                    x[i][0] = x[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (rr < rows && d < hd) {
                        x[i][0] = *reinterpret_cast<const float4*>(qp + d);
                        x[i][1] = *reinterpret_cast<const float4*>(qp + d + 4);
                    }
                }
                if (j0 == 0) vis_fill(vis[r], a, s, b, node);
#pragma unroll
                for (int i = 0; i < UPT; ++i) mb = max(mb, max8(x[i][0], x[i][1]));
#pragma unroll
                for (int o = 1; o < TPR; o <<= 1) mb = max(mb, __shfl_xor_sync(0xFFFFFFFFu, mb, o));
                const int e = half_exponent(mb);
                const float sc = pow2i(-e);
#pragma unroll
                for (int i = 0; i < UPT; ++i) {
                    uint32_t hi[4], lo[4];
                    split8(x[i][0], x[i][1], sc, hi, lo);
                    const uint32_t c = (uint32_t)(j0 + i * TPR);
                    const uint32_t o = (uint32_t)r * (HD * 2) + ((c ^ (r & 7)) << 4);
                    st_shared16(qh + o, hi);
                    st_shared16(ql + o, lo);
                }
                if (j0 == 0) qscale[r] = pow2i(e) * (kLog2e / sqrtf((float)hd));
            }
        }
        if (tid < TREE_MAX_NODES / 32) badrow[tid] = 0;
        if (tid < 4) tmax[tid] = 0;
        if (tid == 0) low = 0;
        __syncthreads();

        float O[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) O[i][0] = O[i][1] = O[i][2] = O[i][3] = 0.f;

#pragma unroll 1
        for (int t = t0; t < t1; ++t) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            const bool tail = (t + 1) * PT > s.n_ctx;
            const uint32_t kh = sb + (KVT == KV_F16 ? (uint32_t)(t & 1) * TN_TILE_BYTES : TN_TILE_BYTES), vh = kh + HALF_TILE;
            const uint32_t mine = KVT == KV_F16 ? own + (uint32_t)(t & 1) * TN_TILE_BYTES : own;
            if (tail) {
                // non-finite values of drafted rows leave the V tile (another row's zero weight
                // must not meet them); rows that see them take them up at the end
#pragma unroll 1
                for (int i = 0; i < NV; ++i) {
                    const uint32_t o = mine + i * OSTEP + HALF_TILE;
                    const int x = t * PT + r0 + i * RSTEP - s.n_ctx;
                    uint4 v = ld_shared16(o);
                    if (x >= 0 && zero_nonfinite<KVT>(v)) {
                        atomicOr(&badrow[x >> 5], 1u << (x & 31));
                        st_shared16(o, {v.x, v.y, v.z, v.w});
                    }
                }
            }
            if (KVT != KV_F16) {
                if (t > t0) __syncthreads();  // the last tile's operands are free
                // split by the last tile's scale; when the values turn out not to fit it
                // (seldom), once more after their own
                for (;;) {
#pragma unroll 1
                    for (int which = 0; which < 2; ++which) {
                        const float f = pow2i(which ? -ev : -ek);
                        const uint32_t dst = which ? vh : kh;
                        uint32_t mb = 0, mn = 0xFFFFFFFFu;
                        uint4 xs[NV];  // (all loads before the first store: the compiler keeps their order)
#pragma unroll
                        for (int i = 0; i < NV; ++i) xs[i] = ld_shared16(mine + i * OSTEP + which * HALF_TILE);
#pragma unroll
                        for (int i = 0; i < NV; ++i) {
                            const int r = r0 + i * RSTEP;
                            const uint4 x = xs[i];
                            const uint32_t top = abs_bits<KVT>(x);
                            mb = max(mb, top);
                            mn = __viaddmin_u32(top, 0xFFFFFFFFu, mn);
                            if (KVT == KV_F32) {
                                uint32_t h0, l0, h1, l1;
                                split2t(__fmul2_rn(make_float2(__uint_as_float(x.x), __uint_as_float(x.y)), make_float2(f, f)), h0, l0);
                                split2t(__fmul2_rn(make_float2(__uint_as_float(x.z), __uint_as_float(x.w)), make_float2(f, f)), h1, l1);
                                const uint32_t o = dst + (uint32_t)r * (HD * 2) + ((((uint32_t)c0 >> 1) ^ (r & 7)) << 4) + (c0 & 1) * 8;
                                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(o), "r"(h0), "r"(h1) : "memory");
                                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(o + F::TILE_H), "r"(l0), "r"(l1) : "memory");
                            } else {
                                uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    w[j] = pack_half2(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xFFFF0000u) * f);
                                st_shared16(dst + (uint32_t)r * (HD * 2) + (((uint32_t)c0 ^ (r & 7)) << 4), w);
                            }
                        }
                        if (__any_sync(0xFFFFFFFFu, mb >= 0x7F800000u)) {  // infinities or NaN: the finite maximum
                            mb = 0;
#pragma unroll 1
                            for (int i = 0; i < NV; ++i) mb = max(mb, max_bits<KVT>(ld_shared16(mine + i * OSTEP + which * HALF_TILE)));
                        }
                        mb = __reduce_max_sync(0xFFFFFFFFu, mb);
                        if (lane == 0) atomicMax(&tmax[2 * (t & 1) + which], mb);
                        if (may_be_low(mn, which ? ev : ek)) low = 1;
                    }
                    __syncthreads();
                    const uint32_t mk = tmax[2 * (t & 1)], mv = tmax[2 * (t & 1) + 1];
                    const bool fk = tile_fits(mk, ek), fv = tile_fits(mv, ev);
                    if (fk && fv) break;
                    if (!fk) ek = tile_exponent(mk);
                    if (!fv) ev = tile_exponent(mv);
                }
                if (tid < 2) tmax[2 * (~t & 1) + tid] = 0;  // the next tile's, last read two barriers ago
            } else {
                __syncthreads();
            }
            if (t + 1 < t1) load(t + 1);
            if (!active) continue;
            const float fk = pow2i(ek), fv = pow2i(ev);
#pragma unroll 1
            for (int pb = 0; pb < F::PW; pb += PB) {
                const int pl0 = wg * F::PW + pb;  // first position of the step in the tile
                // the products of a score's halves in chains of their own, added at the end
                float S[PB / 8][4], S1[PB / 8][4];
#pragma unroll
                for (int i = 0; i < PB / 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) S[i][j] = S1[i][j] = 0.f;
                const int ra = wm * 16 + (lane & 15), ca = lane >> 4, rb = pl0 + (lane & 7) + ((lane >> 4) << 3), cb = (lane >> 3) & 1;
                const uint32_t qrow = (uint32_t)ra * (HD * 2), krow = kh + (uint32_t)rb * (HD * 2);
#pragma unroll 4
                for (int kk = 0; kk < HD / 16; ++kk) {
                    uint32_t ah[4], al[4];
                    const uint32_t oa = qrow + (uint32_t)(((2 * kk + ca) ^ (ra & 7)) << 4);
                    const uint32_t ob = krow + (uint32_t)(((2 * kk + cb) ^ (rb & 7)) << 4);
                    ldsm4(ah, qh + oa);
                    ldsm4(al, ql + oa);
#pragma unroll
                    for (int nb = 0; nb < PB / 16; ++nb) {
                        uint32_t bh[4];
                        ldsm4(bh, ob + nb * 16 * HD * 2);
                        mma16816(S[2 * nb], ah, bh[0], bh[1]);
                        mma16816(S[2 * nb + 1], ah, bh[2], bh[3]);
                        mma16816(S1[2 * nb], al, bh[0], bh[1]);
                        mma16816(S1[2 * nb + 1], al, bh[2], bh[3]);
                        if (NLO == 2) {
                            uint32_t bl[4];
                            ldsm4(bl, ob + nb * 16 * HD * 2 + F::TILE_H);
                            mma16816(S1[2 * nb], ah, bl[0], bl[1]);
                            mma16816(S1[2 * nb + 1], ah, bl[2], bl[3]);
                        }
                    }
                }
                // base-2 scores, masks, running maximum and sum of this thread's two rows
                float alpha[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int r = wm * 16 + g8 + 8 * half;
                    const float f = qscale[r] * fk;
                    // bit i: position i of the step is seen
                    const uint32_t seen = (tail ? vis_window(vis[r], t * PT + pl0 - s.n_ctx) : 0xFFFFFFFFu) >> (2 * q4);
                    float mx = m[half];
#pragma unroll
                    for (int i = 0; i < PB / 8; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float x = (S[i][2 * half + j] + S1[i][2 * half + j]) * f;
                            S[i][2 * half + j] = (seen >> (i * 8 + j)) & 1 ? x : -INFINITY;
                            mx = fmaxf(mx, S[i][2 * half + j]);
                        }
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
                    const float ref = mx == -INFINITY ? 0.f : mx;
                    alpha[half] = exp2_fast(m[half] - ref);
                    m[half] = mx;
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < PB / 8; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float e = exp2_fast(S[i][2 * half + j] - ref + kPShift);
                            S[i][2 * half + j] = e;
                            sum += e;
                        }
                    l[half] = fmaf(l[half], alpha[half], sum);
                }
                // P in two halves (A operand), P V from zero, joined to the running output
                uint32_t ph[PB / 16][4], pq[PB / 16][4];
#pragma unroll
                for (int i = 0; i < PB / 16; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        split2t(make_float2(S[2 * i + (j >> 1)][2 * (j & 1)], S[2 * i + (j >> 1)][2 * (j & 1) + 1]), ph[i][j], pq[i][j]);
                const int rv = pl0 + (lane & 15);
                const uint32_t vrow = vh + (uint32_t)rv * (HD * 2);
#pragma unroll
                for (int db = 0; db < HD / 16; ++db) {
                    float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
                    const uint32_t o = vrow + (uint32_t)(((2 * db + (lane >> 4)) ^ (rv & 7)) << 4);
#pragma unroll
                    for (int i = 0; i < PB / 16; ++i) {
                        uint32_t bh[4];
                        ldsm4t(bh, o + i * 16 * HD * 2);
                        mma16816(d0, ph[i], bh[0], bh[1]);
                        mma16816(d1, ph[i], bh[2], bh[3]);
                        mma16816(d0, pq[i], bh[0], bh[1]);
                        mma16816(d1, pq[i], bh[2], bh[3]);
                        if (NLO == 2) {
                            uint32_t bl[4];
                            ldsm4t(bl, o + i * 16 * HD * 2 + F::TILE_H);
                            mma16816(d0, ph[i], bl[0], bl[1]);
                            mma16816(d1, ph[i], bl[2], bl[3]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        O[2 * db][j] = fmaf(d0[j], fv, O[2 * db][j] * alpha[j >> 1]);
                        O[2 * db + 1][j] = fmaf(d1[j], fv, O[2 * db + 1][j] * alpha[j >> 1]);
                    }
                }
            }
        }
        // the position groups' results meet in shared memory: per row m, l, O
        __syncthreads();
        bool exact = KVT != KV_F16 && low;
        float* fin = reinterpret_cast<float*>(smem);  // [NG][RT][HD + 4]
        if (active) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                l[half] += __shfl_xor_sync(0xFFFFFFFFu, l[half], 1);
                l[half] += __shfl_xor_sync(0xFFFFFFFFu, l[half], 2);
                float* fr = fin + ((size_t)wg * RT + wm * 16 + g8 + 8 * half) * (HD + 4);
#pragma unroll
                for (int i = 0; i < HD / 8; ++i)
                    *reinterpret_cast<float2*>(fr + i * 8 + 2 * q4) = make_float2(O[i][2 * half], O[i][2 * half + 1]);
                if (q4 == 0) {
                    fr[HD] = m[half];
                    fr[HD + 1] = l[half];
                }
            }
        }
        const int anybad = __syncthreads_or(tid < TREE_MAX_NODES / 32 ? badrow[tid] != 0 : 0);
        const bool whole = t0 == 0 && t1 == sg.tiles;
        float* part = parts + ((size_t)blockIdx.x * 2 + (t0 == 0 ? 1 : 0)) * tree_part_floats(RT, hd);
#pragma unroll 1
        for (int i = tid; i < RT * (HD / 4); i += TN_THREADS) {
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4, rr = rtile * RT + r;
            if (rr >= rows || d >= hd) continue;
            const float* fr = fin + (size_t)r * (HD + 4);
            float M = -INFINITY;
#pragma unroll
            for (int g = 0; g < NG; ++g) M = fmaxf(M, fr[(size_t)g * RT * (HD + 4) + HD]);
            const float ref = M == -INFINITY ? 0.f : M;
            float L = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float* fg = fr + (size_t)g * RT * (HD + 4);
                const float w = exp2_fast(fg[HD] - ref);
                const float4 x = *reinterpret_cast<const float4*>(fg + d);
                L = fmaf(fg[HD + 1], w, L);
                o.x = fmaf(x.x, w, o.x);
                o.y = fmaf(x.y, w, o.y);
                o.z = fmaf(x.z, w, o.z);
                o.w = fmaf(x.w, w, o.w);
            }
            const int node = div_rep(rr);
            if (whole) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                float4 y = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
                if (L == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
                *reinterpret_cast<float4*>(a.out + ((size_t)b * a.T + node) * a.ld_out + (size_t)(kvh * rep + rr - node * rep) * hd + d) = y;
            } else {
                *reinterpret_cast<float4*>(part + (size_t)r * hd + d) = o;
                if (d == 0) {
                    part[(size_t)RT * hd + r] = M;
                    part[(size_t)RT * hd + RT + r] = L;
                }
            }
        }
        if (!whole && t0 == 0 && tid == 0)
            desc[blockIdx.x] = TreeDesc{b, kvh, rtile | min(RT, rows - rtile * RT) << 16, sg.last_cta};
        __syncthreads();
        if (KVT != KV_F16 && exact) exact = __syncthreads_or(tree_rows_apart<KVT, PT>(a, sg, warp, TN_THREADS / 32));
        if (KVT != KV_F16 && exact) {
            tree_exact_rows<KVT, PT>(a, sg, RT, rep, &vis[0][0], part, whole, warp, TN_THREADS / 32);
            __syncthreads();
        } else if (anybad) {
            tree_fix_rows<KVT>(a, sg, RT, rep, badrow, &vis[0][0], part, whole, tid, TN_THREADS);
            __syncthreads();
        }
    }
    tree_zero_rows<TN_THREADS>(a);
}

// ---- wide trees: tcgen05, 128 rows per row tile -------------------------------------------------------
// One CTA per SM and range of tiles, sixteen warps:
//   0-7       softmax streams (two warpgroups): even and odd tiles of a segment, a thread per row with
//             a running maximum, sum and output of its own (registers); no shuffles, no exchange
//             until the end;
//   8-11, 14, loaders: a tile is split into f16 halves and written as MMA operands (rows of 64 dims,
//   15        128-byte swizzle): fp32 from raw buffers, bf16 in place, and of either type the last
//             tiles, whose rows may end inside;
//   12        MMA issue;
//   13        copies ahead of the loaders: fp32 rows by bulk copies into raw buffers, bf16 tiles
//             through a tensor map into their operand stages.  (f16 tiles need no loader at all.)
// Tensor memory: S_0, S_1 (PT columns each) and D_0, D_1 (HD columns each).  QK: S_w = Q K^T,
// Q from shared memory, the tile K-major.  The softmax thread overwrites its scores in place,
// CH columns at a time, with the high halves of p (CH / 2 columns) and the low ones, the A
// operand of PV: D_w = P V, the same tile layout read MN-major; D_w starts from zero for every
// tile and joins the registers' output.  QK of tile i + 1 is issued before PV of tile i, so the
// tensor pipe works while a stream is in its softmax.
// 128 positions per tile (64 where fp32 rows of 128 dims would not fit): the costs per tile (waits,
// reductions, the output's join) are spread over most scores.  Registers: HD output sums per softmax
// thread decide the split between the warpgroups.
//
// Bound, 16-bit caches of 64 dims: by the instructions of the two softmax streams, one warp of each
// per scheduler (per 128 x 128 tile about 750 cycles for the maximum, 2700 for exponentials and their
// split, 550 for the join); issue slots 53 %, tensor pipe 38 %, DRAM 35 % of their peaks.  fp32 and
// bf16: by the loaders' split (tensor pipe 16 to 29 %), and for heads of 128 dims by the 22000 cycles
// of a segment's start and end.  Device time, both launches: 32 trees of 64, 8128 positions, 32x8x64
// f16 215 us (342 MB of rows read: 1.6 TB/s; 155 GF in two products: 722 TF/s); 12 trees of 31, 4001
// positions, 32x8x128 bf16 95 us; 1 tree of 64, 16000 positions, 32x8x64 f32 51.4 us (25 GF in three
// products: 490 TF/s).  The look at the range of a tile's rows is 0 to 2 % of that.  A third score buffer (QK two tiles ahead) and chunks of scores fetched ahead
// made no difference and were left out.
constexpr int TW_THREADS = 512;
constexpr int TW_RT = 128;

constexpr int TW_LOADERS = 6;  // loader warps: warpgroup 2 and the last two warps of warpgroup 3

template <int HD, int KVT>
struct WideCfg {
    static constexpr int ESZ = KVT == KV_F32 ? 4 : 2;
    static constexpr int PT = KVT == KV_F32 && HD == 128 ? 64 : 128;
    static constexpr int NLO = KVT == KV_F32 ? 2 : 1;
    static constexpr int HALF = PT * HD * 2;              // bytes of one half of a K or V tile
    static constexpr int RAW = PT * HD * ESZ;             // bytes of a raw fp32 K or V tile
    // operand stages of K and V, raw buffers (fp32)
    static constexpr int KS = KVT == KV_F16 ? (HD == 64 ? 4 : 2) : (KVT == KV_BF16 ? (HD == 64 ? 4 : 2) : 1);
    static constexpr int VS = KVT == KV_F32 ? (HD == 64 ? 2 : 1) : KS;
    static constexpr int RS = 2;
    static constexpr int QH = TW_RT * HD * 2;             // bytes of one half of Q
    static constexpr int Q_OFF = 0;
    static constexpr int K_OFF = 2 * QH;
    static constexpr int V_OFF = K_OFF + KS * NLO * HALF;
    static constexpr int RAW_OFF = V_OFF + VS * NLO * HALF;
    static constexpr int SMEM = RAW_OFF + (KVT == KV_F32 ? RS * RAW : 0) + 1024;
    // registers per thread of the softmax warpgroups and of the other two (512 in all, four
    // warpgroups of 128 at launch)
    static constexpr int REG_S = HD == 64 ? 144 : 192, REG_L = HD == 64 ? 112 : 64;
    static constexpr int CH = HD == 64 ? 32 : 16;         // score columns a softmax thread holds at a time
};

__device__ __forceinline__ uint64_t wide_desc(uint32_t saddr, uint32_t lbo) {
    // start >> 4 [0,14), LBO >> 4 [16,30), SBO >> 4 [32,46) (1024: 8 rows of 128 bytes), version 1
    // [46,48), 128-byte swizzle [61,64)
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// One MMA / commit, issued by the lane whose `lead` is set (elect_lane) while the whole warp runs
// the same code: a warp-uniform loop keeps the descriptors in uniform registers and issues 128 x
// 64 x 16 products every 32 clocks, a loop inside `if (lane == 0)` every 47 to 120.
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void wide_mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(acc), "r"(lead));
}
__device__ __forceinline__ void wide_mma_ts(uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(ta), "l"(db), "r"(idesc), "r"(acc), "r"(lead));
}
__device__ __forceinline__ void wide_commit(uint64_t* bar, uint32_t lead) {
    if (lead)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    __syncwarp();
}
// n columns of a thread's TMEM lane (a load includes its wait)
__device__ __forceinline__ void tmem_ld(uint32_t t, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(t)
                 : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t t, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t t, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(t)
                 : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t t, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int ID, int N>
__device__ __forceinline__ void named_bar() {
    asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory");
}
// byte offset of 16-byte chunk c (8 dims) of row r in a tile of `rows` rows (64-dim blocks)
__device__ __forceinline__ uint32_t wide_off(int rows, int r, int c) {
    return (uint32_t)(c >> 3) * (uint32_t)(rows * 128) + (uint32_t)r * 128u + (uint32_t)(((c & 7) ^ (r & 7)) << 4);
}

struct WideShared {
    // mbarriers, initialised in order by count()
    uint64_t rawfull[8];                          // raw fp32 tiles, bf16 tiles in their operand stages
    uint64_t kfree[4], vfree[4];                  // operand stages: their MMAs are done
    uint64_t sfull[2], dfull[2], done;
    uint64_t kfull[4], vfull[4], rawfree[2];      // one arrival per loader warp
    uint64_t pfull[2], qfull;
    static constexpr int N_BARS = 34;
    __device__ static uint32_t count(int i) { return i < 21 ? 1 : (i < 31 ? TW_LOADERS : (i < 33 ? 128 : 256)); }
    uint32_t tmem;
    int abort;
    unsigned tmax[4];
    int low[8];                                   // by segment: as in the narrow kernel
    int apart;                                    // what is found then
    int ek[8], ev[8];                             // scale exponents of the last eight tiles
    unsigned badrow[8][TREE_MAX_NODES / 32];      // drafted rows with non-finite values, by segment
    float qscale[TW_RT];
    float2 ml[2][TW_RT];                          // the streams' row maxima and sums
    float* dst[TW_RT];                            // where a segment's rows go
    uint32_t vis[256][VIS_WORDS];                 // what each softmax thread's row sees
};

// Half h of a segment's rows from the two streams' staged halves: added, scaled by the row's
// factor (scale[r].x), written coalesced to where dst[r] points (nullptr: not a row).
template <int HD>
__device__ __forceinline__ void wide_rows_out(uint32_t stage, const float2* scale, float* const* dst, int h, int hd) {
    constexpr int LPR = HD / 8, RPW = 32 / LPR, N = TW_RT / RPW / 8, U = 4;  // lanes per half row, rows per warp and step, steps
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane % LPR, d = h * (HD / 2) + c * 4;
#pragma unroll
    for (int k0 = 0; k0 < N; k0 += U) {
        uint4 x[U], y[U];
        float f[U];
        float* to[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int r = (warp + 8 * (k0 + k)) * RPW + lane / LPR;
            const uint32_t at = stage + (uint32_t)r * (HD * 2) + ((uint32_t)(c ^ (r & 7)) << 4);
            x[k] = ld_shared16(at);
            y[k] = ld_shared16(at + TW_RT * HD * 2);
            f[k] = scale[r].x;
            to[k] = dst[r];
        }
#pragma unroll
        for (int k = 0; k < U; ++k)
            // (a row that saw nothing has the factor 0 and zeros; its sum cannot be anything else)
            if (to[k] && d < hd)
                *reinterpret_cast<float4*>(to[k] + d) =
                    make_float4((__uint_as_float(x[k].x) + __uint_as_float(y[k].x)) * f[k], (__uint_as_float(x[k].y) + __uint_as_float(y[k].y)) * f[k],
                                (__uint_as_float(x[k].z) + __uint_as_float(y[k].z)) * f[k], (__uint_as_float(x[k].w) + __uint_as_float(y[k].w)) * f[k]);
    }
}
__device__ __forceinline__ bool badrow_any(const unsigned* badrow) {
    unsigned v = 0;
#pragma unroll
    for (int w = 0; w < TREE_MAX_NODES / 32; ++w) v |= badrow[w];
    return v != 0;
}

template <int HD, int KVT>
__global__ void __launch_bounds__(TW_THREADS, 1)
    tf_tree_attn_wide_kernel(const __grid_constant__ TreeAttnArgs a, const __grid_constant__ TreePlan pl,
                             const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using F = WideCfg<HD, KVT>;
    constexpr int PT = F::PT, NLO = F::NLO, ESZ = F::ESZ, KS = F::KS, VS = F::VS, RS = F::RS, CH = F::CH;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(16) WideShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
    const int rep = pl.rep, hd = a.hd;
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    volatile int* abort_flag = &sh.abort;
    const int rep_inv = pl.rep_inv;

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    if (tid == 32) {
#pragma unroll 1
        for (int i = 0; i < WideShared::N_BARS; ++i) mbar_init(&sh.rawfull[i], WideShared::count(i));
        sh.abort = 0;
        mbar_fence_init();
    }
    if (tid < 4) sh.tmax[tid] = 0;
    pdl_trigger();
    pdl_wait();
    TreeDesc* desc = static_cast<TreeDesc*>(a.ws);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + 65536);
    if (tid == 0) desc[blockIdx.x].b = -1;
    TreeIter it;
    tree_range<PT, TW_RT, TW_UNIT_COST>(a, pl, it);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    TreeSeg sg;

    // Every role walks the same segments and tiles; after an abort the waits return at once and
    // the roles run on without effect, so that all of them meet at every barrier.
    // A 16-bit tile of committed context comes straight to its operand stage through the tensor
    // maps: f16 is done then, bf16 is converted in place.  The last tiles of a sequence (drafted
    // rows, the end of the cache) are fetched by the loaders' own loads.
    auto direct = [&](const TreeSeg& g, int t) { return KVT != KV_F32 && pl.maps && (t + 1) * PT <= g.s.n_ctx; };
    auto tma_tile = [&](const TreeSeg& g, int t, int which, uint32_t off, uint64_t* bar) {
        mbar_expect_tx(bar, F::HALF);
        const int row = g.s.slot * pl.slot_rows + g.kvh * a.cap + t * PT;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
            asm volatile(
                "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                    sb + off + c * PT * 128),
                "l"(reinterpret_cast<uint64_t>(which ? &vmap : &kmap)), "r"(64 * c), "r"(row), "r"(smem_u32(bar))
                : "memory");
    };
    if (wg >= 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::REG_L));
    if (wg == 2 || warp >= 14) {
        constexpr int LT = TW_LOADERS * 32;
        const int lt = wg == 2 ? tid - 256 : tid - 320;
        int n = 0, nr = 0, nd = 0, seg = 0;  // running tile, raw buffer, direct tile, segment
        constexpr int VPR = HD * ESZ / 16, RSTEP = LT / VPR;  // 16-byte vectors per row, rows per step of all loaders
        constexpr int UNR = 6;               // vectors in flight per thread
        int ek = TILE_FIRST, ev = TILE_FIRST;  // scale exponents of K and V, kept from tile to tile
        const int r0 = lt / VPR, c0 = lt % VPR;
        // where this thread's vectors of a whole tile go: row r0 + k * RSTEP at rel[k % NB] + k * RSTEP * 128
        // (the swizzle depends on the row modulo 8)
        constexpr int NVT = (PT + RSTEP - 1) / RSTEP, NB = RSTEP % 8 == 0 ? 1 : (RSTEP % 4 == 0 ? 2 : 4);
        // the vector of row lt that this thread looks at (fp32: from the thread's first one on)
        const int look_c = lt % (hd * ESZ / 16), look = lt * hd * 4 + look_c * 16 - (r0 * hd * 4 + c0 * 16);
        uint32_t rel[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int c = KVT == KV_F32 ? c0 >> 1 : c0;
            rel[j] = wide_off(PT, r0, c) - (uint32_t)(((c & 7) ^ (r0 & 7)) << 4) + (uint32_t)(((c & 7) ^ ((r0 + j * RSTEP) & 7)) << 4) +
                     (KVT == KV_F32 ? (c0 & 1) * 8 : 0);
        }
        while (tree_next<PT, TW_RT, TW_UNIT_COST>(a, rep, it, sg)) {
            const TreeSeq s = sg.s;
            if (lt < TREE_MAX_NODES / 32) sh.badrow[seg & 7][lt] = 0;  // read by others long ago
            if (lt == 0) sh.low[seg & 7] = 0;
            named_bar<2, LT>();
#pragma unroll 1
            for (int t = sg.t0; t < sg.t1; ++t, ++n) {
                const int rows = min(PT, s.n_ctx + s.n_node - t * PT);
                const bool dir = direct(sg, t), tail = (t + 1) * PT > s.n_ctx;
#pragma unroll 1
                for (int which = 0; which < 2; ++which) {
                    const int st = which ? VS : KS, os = n % st;
                    uint64_t* full = which ? &sh.vfull[os] : &sh.kfull[os];
                    uint64_t* free = which ? &sh.vfree[os] : &sh.kfree[os];
                    const uint32_t off = which ? F::V_OFF + os * NLO * F::HALF : F::K_OFF + os * NLO * F::HALF;
                    const uint32_t dst = sb + off;
                    // the operand stage is free once the MMAs of its last tile are done (every loader
                    // waits for every tile: a wait tells a phase from its neighbours only)
                    if (n >= st) tree_wait(free, n / st - 1, a.err, ERR_WAIT_EMPTY, abort_flag);
                    __syncwarp();
                    if (KVT == KV_F16 && dir) {
                        if (lane == 0) {
                            if (lt == 0 && !*abort_flag) tma_tile(sg, t, which, off, full);
                            else mbar_arrive(full);
                        }
                        __syncwarp();
                        continue;
                    }
                    uint32_t src = 0;  // this thread's first vector in shared memory, rows sstep bytes apart
                    if (KVT == KV_F32) {
                        const int rs = nr % RS;
                        src = sb + F::RAW_OFF + rs * F::RAW + (uint32_t)(r0 * hd * 4 + c0 * 16);
                        tree_wait(&sh.rawfull[rs], nr / RS, a.err, ERR_WAIT_FULL, abort_flag);
                    } else if (dir) {
                        tree_wait(&sh.rawfull[(nd & 3) * 2 + which], nd >> 2, a.err, ERR_WAIT_FULL, abort_flag);
                    } else {  // from the cache to the operand's place
                        const uint8_t* g = static_cast<const uint8_t*>(which ? a.vc : a.kc) +
                                           ((size_t)s.slot * a.slot_stride + ((size_t)sg.kvh * a.cap + (size_t)t * PT) * hd + c0 * 8) * 2;
#pragma unroll 4
                        for (int r = r0; r < PT; r += RSTEP) {
                            uint4 x = make_uint4(0, 0, 0, 0);
                            if (r < rows && c0 * 8 < hd) x = *reinterpret_cast<const uint4*>(g + (size_t)r * hd * 2);
                            st_shared16(dst + wide_off(PT, r, c0), {x.x, x.y, x.z, x.w});
                        }
                    }
                    __syncwarp();
                    if (KVT == KV_F32 && rows < PT)  // rows behind the end are zeros
#pragma unroll 1
                        for (int r = r0; r < PT; r += RSTEP)
                            if (r >= rows) st_shared16(src + (uint32_t)((r - r0) * hd * 4), {0u, 0u, 0u, 0u});
                    const bool col = KVT != KV_F32 || c0 * 4 < hd;
                    auto at = [&](int r) { return KVT == KV_F32 ? src + (uint32_t)((r - r0) * hd * 4) : dst + wide_off(PT, r, c0); };
                    if (which && tail && col) {  // non-finite drafted values leave the operand (see the narrow kernel)
#pragma unroll 1
                        for (int r = r0; r < rows; r += RSTEP) {
                            const int p = t * PT + r - s.n_ctx;
                            if (p < 0) continue;
                            uint4 x = ld_shared16(at(r));
                            if (zero_nonfinite<KVT>(x)) {
                                atomicOr(&sh.badrow[seg & 7][p >> 5], 1u << (p & 31));
                                st_shared16(at(r), {x.x, x.y, x.z, x.w});
                            }
                        }
                    }
                    if (KVT != KV_F16) {
                        // split by the last tile's scale; when the values turn out not to fit it
                        // (seldom), once more after their own.  bf16 tiles are converted in place, so
                        // their range is found first.
                        unsigned* tm = &sh.tmax[2 * (n & 1) + which];
                        // a whole tile's vectors lie at compile-time distances; this thread's last one
                        // may not exist
                        const bool whole_tile = hd == HD, has_last = r0 + (NVT - 1) * RSTEP < PT;
                        uint32_t place[NB];
#pragma unroll
                        for (int j = 0; j < NB; ++j) place[j] = dst + rel[j];
                        auto from = [&](int k) { return KVT == KV_F32 ? src + (uint32_t)(k * RSTEP * HD * 4) : place[k % NB] + (uint32_t)(k * RSTEP * 128); };
                        auto split_store = [&](const uint4& x, float2 f, uint32_t o) {  // fp32 halves
                            uint32_t h0, l0, h1, l1;
                            split2t(__fmul2_rn(make_float2(__uint_as_float(x.x), __uint_as_float(x.y)), f), h0, l0);
                            split2t(__fmul2_rn(make_float2(__uint_as_float(x.z), __uint_as_float(x.w)), f), h1, l1);
                            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(o), "r"(h0), "r"(h1) : "memory");
                            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(o + F::HALF), "r"(l0), "r"(l1) : "memory");
                        };
                        auto half_store = [&](const uint4& x, float2 f, uint32_t o) {  // bf16 in one half
                            uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float2 y = __fmul2_rn(make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u)), f);
                                w[j] = pack_half2(y.x, y.y);
                            }
                            st_shared16(o, w);
                        };
                        if (KVT == KV_F32 ? tail : !dir) named_bar<2, LT>();  // (the others' stores, for the look at a row)
                        for (;;) {
                            const int e = which ? ev : ek;
                            const float2 f = make_float2(pow2i(-e), pow2i(-e));
                            uint32_t mb = 0;
                            // one vector of a row, a row per thread, tells most tiles whose rows share a scale
                            if (lt < rows && may_be_low(abs_bits<KVT>(ld_shared16(KVT == KV_F32 ? src + look : dst + wide_off(PT, lt, look_c))), e))
                                sh.low[seg & 7] = 1;
                            if (whole_tile) {
#pragma unroll
                                for (int k0 = 0; k0 < NVT; k0 += UNR) {  // (all loads before the first store: the compiler keeps their order)
                                    uint4 x[UNR];
#pragma unroll
                                    for (int k = k0; k < k0 + UNR && k < NVT; ++k) {
                                        x[k - k0] = make_uint4(0, 0, 0, 0);
                                        if (k < NVT - 1 || has_last) x[k - k0] = ld_shared16(from(k));
                                    }
#pragma unroll
                                    for (int k = k0; k < k0 + UNR && k < NVT; ++k) {
                                        abs_max<KVT>(mb, x[k - k0]);
                                        if (KVT == KV_F32 && (k < NVT - 1 || has_last))
                                            split_store(x[k - k0], f, place[k % NB] + (uint32_t)(k * RSTEP * 128));
                                    }
                                }
                                mb = abs_max_bits<KVT>(mb);
                            } else {
#pragma unroll 1
                                for (int r = r0; r < PT; r += RSTEP) {
                                    uint4 x = make_uint4(0, 0, 0, 0);
                                    if (r < rows && col) x = ld_shared16(at(r));
                                    mb = max(mb, abs_bits<KVT>(x));
                                    if (KVT == KV_F32) split_store(x, f, dst + wide_off(PT, r, c0 >> 1) + (c0 & 1) * 8);
                                }
                            }
                            if (__any_sync(0xFFFFFFFFu, mb >= 0x7F800000u)) {  // infinities or NaN: the finite maximum
                                mb = 0;
                                if (col)
#pragma unroll 1
                                    for (int r = r0; r < rows; r += RSTEP) mb = max(mb, max_bits<KVT>(ld_shared16(at(r))));
                                __syncwarp();
                            }
                            mb = __reduce_max_sync(0xFFFFFFFFu, mb);
                            if (lane == 0) atomicMax(tm, mb);
                            named_bar<2, LT>();
                            const uint32_t all = *tm;
                            if (tile_fits(all, e)) break;
                            (which ? ev : ek) = tile_exponent(all);
                            named_bar<2, LT>();  // (the maximum is read by all before it is raised again)
                        }
                        if (lt == 0) {
                            sh.tmax[2 * (~n & 1) + which] = 0;  // the next tile's, read last a tile ago
                            (which ? sh.ev : sh.ek)[n & 7] = which ? ev : ek;
                        }
                        if (KVT == KV_BF16) {
                            const float2 f = make_float2(pow2i(which ? -ev : -ek), pow2i(which ? -ev : -ek));
                            if (whole_tile) {
#pragma unroll
                                for (int k0 = 0; k0 < NVT; k0 += UNR) {
                                    uint4 x[UNR];
#pragma unroll
                                    for (int k = k0; k < k0 + UNR && k < NVT; ++k) {
                                        x[k - k0] = make_uint4(0, 0, 0, 0);
                                        if (k < NVT - 1 || has_last) x[k - k0] = ld_shared16(from(k));
                                    }
#pragma unroll
                                    for (int k = k0; k < k0 + UNR && k < NVT; ++k)
                                        if (k < NVT - 1 || has_last) half_store(x[k - k0], f, from(k));
                                }
                            } else {
#pragma unroll 1
                                for (int r = r0; r < PT; r += RSTEP) half_store(ld_shared16(at(r)), f, at(r));
                            }
                        }
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(full);
                        if (KVT == KV_F32) mbar_arrive(&sh.rawfree[nr % RS]);
                    }
                    ++nr;
                }
                if (KVT == KV_BF16 && dir) ++nd;
            }
            ++seg;
        }
        // after an abort: copies of the last stages may still be on their way
        if (KVT == KV_F16 && lt == 0 && *abort_flag)
#pragma unroll 1
            for (int i = max(0, n - KS); i < n; ++i) {
                tree_wait(&sh.kfull[i % KS], i / KS, a.err, ERR_WAIT_FULL, nullptr);
                tree_wait(&sh.vfull[i % KS], i / KS, a.err, ERR_WAIT_FULL, nullptr);
            }
    } else if (warp == 13) {
        // copies ahead of the loaders: raw fp32 tiles, bf16 tiles into their operand stages
        if (KVT != KV_F16 && lane == 0) {
            int n = 0, nr = 0, nd = 0;
            unsigned issued = 0, par = 0;  // per barrier: a copy was issued, parity of the last one
            while (tree_next<PT, TW_RT, TW_UNIT_COST>(a, rep, it, sg))
#pragma unroll 1
                for (int t = sg.t0; t < sg.t1; ++t, ++n)
#pragma unroll 1
                    for (int which = 0; which < 2; ++which) {
                        const bool dir = direct(sg, t);
                        int bar, phase;
                        if (KVT == KV_F32) {
                            const int rs = nr % RS;
                            if (nr >= RS) tree_wait(&sh.rawfree[rs], nr / RS - 1, a.err, ERR_WAIT_EMPTY, abort_flag);
                            bar = rs;
                            phase = nr / RS;
                        } else {
                            // every tile's stage is waited for, the loaders' own tiles among them
                            const int os = n % KS;
                            if (n >= KS) tree_wait(which ? &sh.vfree[os] : &sh.kfree[os], n / KS - 1, a.err, ERR_WAIT_EMPTY, abort_flag);
                            bar = (nd & 3) * 2 + which;
                            phase = nd >> 2;
                        }
                        ++nr;
                        if (!*abort_flag && (KVT == KV_F32 || dir)) {
                            if (KVT == KV_F32) {
                                const uint32_t bytes = (uint32_t)(min(PT, sg.s.n_ctx + sg.s.n_node - t * PT) * hd * ESZ);
                                const size_t off = ((size_t)sg.s.slot * a.slot_stride + ((size_t)sg.kvh * a.cap + (size_t)t * PT) * hd) * ESZ;
                                mbar_expect_tx(&sh.rawfull[bar], bytes);
                                bulk_g2s(smem + F::RAW_OFF + bar * F::RAW, static_cast<const uint8_t*>(which ? a.vc : a.kc) + off, bytes,
                                         &sh.rawfull[bar]);
                            } else {
                                tma_tile(sg, t, which, (which ? F::V_OFF : F::K_OFF) + (n % KS) * F::HALF, &sh.rawfull[bar]);
                            }
                            issued |= 1u << bar;
                            par = (par & ~(1u << bar)) | ((unsigned)(phase & 1) << bar);
                        }
                        if (which && dir) ++nd;
                    }
            if (*abort_flag)  // copies that may still be on their way
#pragma unroll 1
                for (int i = 0; i < 8; ++i)
                    if (issued >> i & 1) tree_wait(&sh.rawfull[i], par >> i & 1, a.err, ERR_WAIT_FULL, nullptr);
        }
        __syncwarp();
    } else if (warp == 12) {
        // D f32, A / B f16, M = 128: QK with N = PT, both K-major; PV with N = HD, B MN-major
        constexpr uint32_t iqk = (1u << 4) | ((uint32_t)(PT >> 3) << 17) | ((uint32_t)(TW_RT >> 4) << 24);
        constexpr uint32_t ipv = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(TW_RT >> 4) << 24);
        const uint32_t lead = elect_lane(), tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        int n = 0, seg = 0, cnt[2] = {0, 0};  // running tile, segment, PVs issued per stream
        bool ok = true;
        auto wait = [&](uint64_t* bar, int parity) {
            ok = __all_sync(0xFFFFFFFFu, ok && tree_wait(bar, parity, a.err, ERR_WAIT_FULL, abort_flag));
        };
        while (tree_next<PT, TW_RT, TW_UNIT_COST>(a, rep, it, sg)) {
            wait(&sh.qfull, seg);
            // QK of tile t, then PV of tile t - 1 (one step more than there are tiles)
#pragma unroll 1
            for (int t = sg.t0; t <= sg.t1; ++t) {
                const int w = (t - sg.t0) & 1;
                if (t < sg.t1) {
                    const int os = n % KS;
                    wait(&sh.kfull[os], n / KS);
                    if (ok) {
                        tc_fence_after();
                        const uint32_t d = tm + w * 128;
                        const uint64_t kb = wide_desc(sb + F::K_OFF + os * NLO * F::HALF, 16), qb = wide_desc(sb + F::Q_OFF, 16);
                        // the products with a low half first: each step truncates at the size of the
                        // sum so far, which the high halves' products bring up only then
#pragma unroll
                        for (int hi = 0; hi < 2; ++hi)
#pragma unroll
                            for (int j = 0; j < HD / 16; ++j) {  // 16 dims: 32 bytes along the rows of a 64-dim block
                                const uint64_t q = qb + ((j / 4) * (TW_RT * 128) + (j % 4) * 32) / 16;
                                const uint64_t k = kb + ((j / 4) * (PT * 128) + (j % 4) * 32) / 16;
                                wide_mma_ss(d, hi ? q : q + F::QH / 16, k, iqk, hi || j > 0, lead);
                                if (NLO == 2 && !hi) wide_mma_ss(d, q, k + F::HALF / 16, iqk, 1, lead);
                            }
                        wide_commit(&sh.kfree[os], lead);
                        wide_commit(&sh.sfull[w], lead);
                    }
                    ++n;
                }
                if (t > sg.t0) {
                    const int mt = t < sg.t1 ? n - 2 : n - 1, v = w ^ 1, os = mt % VS;  // tile, stream, stage
                    wait(&sh.pfull[v], v ? cnt[1] : cnt[0]);
                    wait(&sh.vfull[os], mt / VS);
                    if (v) ++cnt[1];
                    else ++cnt[0];
                    if (ok) {
                        tc_fence_after();
                        const uint32_t d = tm + 256 + v * HD, p = tm + v * 128;
                        const uint64_t vh = wide_desc(sb + F::V_OFF + os * NLO * F::HALF, PT * 128);
#pragma unroll
                        for (int hi = 0; hi < 2; ++hi)
#pragma unroll
                            for (int j = 0; j < PT / 16; ++j) {  // 16 positions: 2048 bytes of rows; p's halves in blocks of CH columns
                                const uint32_t ph = CH == 32 ? p + 32 * (j / 2) + 8 * (j % 2) : p + 16 * j;
                                wide_mma_ts(d, hi ? ph : ph + CH / 2, vh + 128u * j, ipv, hi || j > 0, lead);
                                if (NLO == 2 && !hi) wide_mma_ts(d, ph, vh + F::HALF / 16 + 128u * j, ipv, 1, lead);
                            }
                        wide_commit(&sh.vfree[os], lead);
                        wide_commit(&sh.dfull[v], lead);
                    }
                }
            }
            ++seg;
        }
        wide_commit(&sh.done, lead);  // arrives once every MMA issued above has completed
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F::REG_S));
        const int row = tid & 127;                                  // TMEM lane
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t ts = tl + wg * 128, td = tl + 256 + wg * HD;
        int n = 0, seg = 0, cnt = 0;
        while (tree_next<PT, TW_RT, TW_UNIT_COST>(a, rep, it, sg)) {
            const TreeSeq s = sg.s;
            const int rows = s.n_node * rep;
            {   // queries, HD / 8 lanes per row: scaled to [2^14, 2^15), two halves
                constexpr int LPR = HD / 8, RPW = 32 / LPR, STEPS = TW_RT / (8 * RPW), U = STEPS;
                const int c = lane % LPR;
                const float* qb = a.q + (size_t)sg.b * a.T * a.ld_q + (size_t)sg.kvh * rep * hd + c * 8;
                const float qk = kLog2e / sqrtf((float)hd);
#pragma unroll 1
                for (int i0 = 0; i0 < STEPS; i0 += U) {
                    float4 x[U][2];
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        const int r = ((i0 + i) * 8 + warp) * RPW + lane / LPR, q = sg.rtile * TW_RT + r, nd = (q * rep_inv) >> 16;
                        const float* qp = qb + ((long long)nd * a.ld_q + (q - nd * rep) * hd);
                        x[i][0] = x[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (q < rows && c * 8 < hd) {
                            x[i][0] = reinterpret_cast<const float4*>(qp)[0];
                            x[i][1] = reinterpret_cast<const float4*>(qp)[1];
                        }
                    }
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        const int r = ((i0 + i) * 8 + warp) * RPW + lane / LPR;
                        uint32_t mb = max8(x[i][0], x[i][1]);
#pragma unroll
                        for (int o = 1; o < LPR; o <<= 1) mb = max(mb, __shfl_xor_sync(0xFFFFFFFFu, mb, o));
                        const int e = half_exponent(mb);
                        uint32_t hi[4], lo[4];
                        split8(x[i][0], x[i][1], pow2i(-e), hi, lo);
                        const uint32_t o = sb + F::Q_OFF + wide_off(TW_RT, r, c);
                        st_shared16(o, hi);
                        st_shared16(o + F::QH, lo);
                        if (c == 0) sh.qscale[r] = pow2i(e) * qk;
                    }
                }
                fence_async();
                mbar_arrive(&sh.qfull);
                named_bar<1, 256>();
            }
            const float qs = sh.qscale[row];
            const int rr = sg.rtile * TW_RT + row, node = (rr * rep_inv) >> 16;
            uint32_t* vis = sh.vis[tid];
            vis_fill(vis, a, s, sg.b, node);
            float O[HD], m = -INFINITY, l = 0.f;
#pragma unroll
            for (int i = 0; i < HD; ++i) O[i] = 0.f;
            const int n0 = n - sg.t0;
#pragma unroll 1
            for (int t = sg.t0 + wg; t < sg.t1; t += 2, ++cnt) {
                tree_wait(&sh.sfull[wg], cnt, a.err, ERR_WAIT_FULL, abort_flag);
                __syncwarp();
                tc_fence_after();
                // (not below the smallest normal number: a query of zeros over small keys would make it zero, and
                // the masked scores' -infinity a NaN; scores that small are equal)
                const float f = KVT == KV_F16 ? qs : fmaxf(qs * pow2i(sh.ek[(n0 + t) & 7]), 1.17549435e-38f);
                const bool tail = (t + 1) * PT > s.n_ctx;
                // (the loops over CH-column chunks stay loops: unrolled, the code outgrows the
                // instruction cache and the one warp per scheduler waits for its fetches)
                float mx = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < PT; c += CH) {
                    uint32_t x[CH];
                    tmem_ld(ts + c, x);
                    if (tail) {
                        const uint32_t seen = vis_window(vis, t * PT + c - s.n_ctx);
#pragma unroll
                        for (int i = 0; i < CH; ++i) x[i] = (seen >> i) & 1 ? x[i] : 0xFF800000u;
                        __syncwarp();
                        tmem_st(ts + c, x);  // masked scores are -infinity from here on
                    }
                    float m0 = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
#pragma unroll
                    for (int i = 2; i < CH; i += 2) m0 = fmaxf(m0, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
                    mx = fmaxf(mx, m0);
                }
                if (tail) tmem_wait_st();
                mx = fmaxf(m, mx * f);
                const float ref = mx == -INFINITY ? 0.f : mx, alpha = exp2_fast(m - ref), shift = kPShift - ref;
                m = mx;
                float sum0 = 0.f, sum1 = 0.f;
#pragma unroll 1
                for (int c = 0; c < PT; c += CH) {
                    uint32_t x[CH], y[CH];
                    tmem_ld(ts + c, x);
#pragma unroll
                    for (int i = 0; i < CH; i += 2) {
                        const float p0 = exp2_fast(fmaf(__uint_as_float(x[i]), f, shift));
                        const float p1 = exp2_fast(fmaf(__uint_as_float(x[i + 1]), f, shift));
                        sum0 += p0;
                        sum1 += p1;
                        split2t(make_float2(p0, p1), y[i / 2], y[CH / 2 + i / 2]);
                    }
                    tmem_st(ts + c, y);
                }
                l = fmaf(l, alpha, sum0 + sum1);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&sh.pfull[wg]);
                tree_wait(&sh.dfull[wg], cnt, a.err, ERR_WAIT_FULL, abort_flag);
                __syncwarp();
                tc_fence_after();
                const float fv = KVT == KV_F16 ? 1.f : pow2i(sh.ev[(n0 + t) & 7]);
#pragma unroll
                for (int c = 0; c < HD / CH; ++c) {
                    uint32_t x[CH];
                    tmem_ld(td + CH * c, x);
#pragma unroll
                    for (int i = 0; i < CH; i += 2) {
                        const float2 o = __ffma2_rn(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), make_float2(fv, fv),
                                                    __fmul2_rn(make_float2(O[CH * c + i], O[CH * c + i + 1]), make_float2(alpha, alpha)));
                        O[CH * c + i] = o.x;
                        O[CH * c + i + 1] = o.y;
                    }
                }
                tc_fence_before();
            }
            n += sg.t1 - sg.t0;
            // The streams meet in Q's shared memory (every QK of the segment is done), half of the
            // columns at a time: both leave their rows weighted, then all threads add the two,
            // divide, and write coalesced.  fp32 rows of HD / 2 per stream, 16-byte chunk c of row
            // r at c ^ (r & 7).
            sh.ml[wg][row] = make_float2(m, l);
            named_bar<1, 256>();
            const bool whole = sg.t0 == 0 && sg.t1 == sg.tiles;
            float* part = parts + ((size_t)blockIdx.x * 2 + (sg.t0 == 0 ? 1 : 0)) * tree_part_floats(TW_RT, hd);
            float wgt;
            {
                const float2 other = sh.ml[wg ^ 1][row];
                const float M = fmaxf(m, other.x), mref = M == -INFINITY ? 0.f : M;
                wgt = exp2_fast(m - mref);
                const float L = fmaf(l, wgt, other.y * exp2_fast(other.x - mref));
                named_bar<1, 256>();
                if (wg == 0) {
                    float* to = whole ? a.out + ((size_t)sg.b * a.T + node) * a.ld_out + (size_t)(sg.kvh * rep + rr - node * rep) * hd
                                      : part + (size_t)row * hd;
                    sh.dst[row] = rr < rows && !*abort_flag ? to : nullptr;
                    sh.ml[0][row].x = !whole ? 1.f : (L == 0.f ? 0.f : 1.f / L);
                    if (!whole && rr < rows && !*abort_flag) {
                        part[(size_t)TW_RT * hd + row] = M;
                        part[(size_t)TW_RT * hd + TW_RT + row] = L;
                    }
                }
            }
            constexpr int HC = HD / 8;  // 16-byte chunks of half a row
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t srow = sb + F::Q_OFF + (uint32_t)wg * (TW_RT * HD * 2) + (uint32_t)row * (HD * 2);
#pragma unroll
                for (int c = 0; c < HC; ++c) {
                    const int i = h * (HD / 2) + 4 * c;
                    st_shared16(srow + ((uint32_t)(c ^ (row & 7)) << 4),
                                {__float_as_uint(O[i] * wgt), __float_as_uint(O[i + 1] * wgt), __float_as_uint(O[i + 2] * wgt),
                                 __float_as_uint(O[i + 3] * wgt)});
                }
                named_bar<1, 256>();
                wide_rows_out<HD>(sb + F::Q_OFF, sh.ml[0], sh.dst, h, hd);
                named_bar<1, 256>();  // the shared memory takes the next half, or the next segment's queries
            }
            if (!whole && sg.t0 == 0 && tid == 0)
                desc[blockIdx.x] =
                    TreeDesc{sg.b, sg.kvh, sg.rtile | min(TW_RT, sg.s.n_node * rep - sg.rtile * TW_RT) << 16, sg.last_cta};
            bool exact = KVT != KV_F16 && sh.low[seg & 7];
            if (KVT != KV_F16 && exact) {
                if (tid == 0) sh.apart = 0;
                named_bar<1, 256>();
                if (tree_rows_apart<KVT, PT>(a, sg, warp, 8)) sh.apart = 1;
                named_bar<1, 256>();
                exact = sh.apart;
            }
            if (KVT != KV_F16 && exact) {
                if (!*abort_flag) tree_exact_rows<KVT, PT>(a, sg, TW_RT, rep, &sh.vis[0][0], part, whole, warp, 8);
                named_bar<1, 256>();
            } else if (badrow_any(sh.badrow[seg & 7])) {
                if (!*abort_flag)
                    tree_fix_rows<KVT>(a, sg, TW_RT, rep, sh.badrow[seg & 7], &sh.vis[0][0], part, whole, tid, 256);
                named_bar<1, 256>();  // (its reads of vis end before the next segment's)
            }
            __syncwarp();
            ++seg;
        }
    }
    // TMEM stays allocated until every issued MMA has completed
    __syncwarp();
    if (warp == 0) tree_wait(&sh.done, 0, a.err, ERR_WAIT_FULL, nullptr);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    tree_zero_rows<TW_THREADS>(a);
}

// ---- joins the partial results of units that were split over CTAs ------------------------------------
// Block (c, y): the unit that starts in CTA c's range and ends in a later one; a warp per row.
// out = sum_i w_i o_i / sum_i w_i l_i, w_i = exp2(m_i - max m).  Bound by the latency of its loads
// (descriptor; maxima and sums; rows): eight rows in flight took 15.2 us of a tree of 5 at 1733
// positions to 12.7, and 35.2 us of one of 9 at 16000 to 25.4.
constexpr int TC_THREADS = 256;
__global__ void __launch_bounds__(TC_THREADS) tf_tree_combine_kernel(const TreeAttnArgs a, const TreePlan pl) {
    pdl_trigger();
    pdl_wait();
    const int c0 = blockIdx.x, lane = threadIdx.x & 31;
    const int r = blockIdx.y * (TC_THREADS / 32) + (threadIdx.x >> 5);
    const TreeDesc de = static_cast<const TreeDesc*>(a.ws)[c0];
    if (de.b < 0 || r >= de.tile >> 16) return;
    const float* parts = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.ws) + 65536);
    const int rep = a.n_head / a.n_kv, hd = a.hd, rt = pl.rt, n = de.c1 - c0 + 1;
    const int rr = (de.tile & 0xFFFF) * rt + r;
    const size_t pf = tree_part_floats(rt, hd);
    auto part = [&](int i) { return parts + ((size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * pf; };
    // 32 parts at a time, a lane per part for the weights and per four dims for the sums; eight
    // parts' loads in flight
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const int d = lane * 4;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int k = min(32, n - i0);
        float m = -INFINITY, l = 0.f;
        if (lane < k) {
            const float* p = part(i0 + lane) + (size_t)rt * hd + r;
            m = p[0];
            l = p[rt];
        }
        float w = 0.f;
#pragma unroll 1
        for (int i = 0; i < k; i += 8) {
            float4 x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = i + j < k && d < hd ? *reinterpret_cast<const float4*>(part(i0 + i + j) + (size_t)r * hd + d)
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
            if (i == 0) {
                const float mx = fmaxf(M, warp_max(m)), ref = mx == -INFINITY ? 0.f : mx, alpha = exp2_fast(M - ref);
                M = mx;
                w = exp2_fast(m - ref);
                L = fmaf(L, alpha, warp_sum(l * w));
                o = make_float4(o.x * alpha, o.y * alpha, o.z * alpha, o.w * alpha);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float wi = __shfl_sync(0xFFFFFFFFu, w, i + j);
                o.x = fmaf(x[j].x, wi, o.x);
                o.y = fmaf(x[j].y, wi, o.y);
                o.z = fmaf(x[j].z, wi, o.z);
                o.w = fmaf(x[j].w, wi, o.w);
            }
        }
    }
    if (d < hd) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const float4 y = L == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        *reinterpret_cast<float4*>(a.out + ((size_t)de.b * a.T + rr / rep) * a.ld_out + (size_t)(de.kvh * rep + rr % rep) * hd + d) = y;
    }
}

// ---- host ------------------------------------------------------------------------------------------
constexpr int TA_MAX_GRID = 1024;  // descriptors of 16 bytes in the workspace's first 64 KB (grid <= 2 CTAs per SM)

static int tree_sms() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms < 1 ? 1 : (2 * sms > TA_MAX_GRID ? TA_MAX_GRID / 2 : sms);
}

// Rows of a unit's row tile, which chooses the kernel too: TW_RT the wide one, fewer the narrow one.
// Device time, narrow / wide (f32 unless said; B trees of T nodes, positions, heads x kv heads x dims),
// measured before the look at the rows' range, which costs the narrow kernel 1 to 4 % and the wide
// one 0 to 2 %:
//   17 to 32 rows:   1 x 8, 100, 32x8x64: 10.4 / 19.3 us;  32 x 8, 1144, 32x8x64 f16: 34.1 / 42.3;
//                    the same in f32: 61.9 / 60.7;  1 x 8, 8000: 22.9 / 22.8
//   33 to 64 rows:   1 x 12, 100, 32x8x64 (0.4 MB of K and V): 12.8 / 19.2;  1 x 5, 1733, 14x2x64
//                    (1.8 MB): 12.7 / 15.2;  2 x 14, 700, 32x8x64 f16 (2.9 MB): 14.3 / 14.0;
//                    1 x 9, 2000, 12x2x128 (4.1 MB): 17.8 / 18.6;  32 x 8, 1144, 12x2x128: 39.1 /
//                    37.1;  32 x 10, 1144, 32x8x64: 59.1 / 52.1;  16 x 12, 4000, in f16: 50.1 / 40.3
//   the same, 16-bit rows of 128 dims (12x2x128, f16; bf16; positions):  1 x 9, 2000: 16.3 / 16.7;
//                    18.2 / 21.7;  32 x 8, 1144: 25.1 / 29.2; 29.2 / 40.3;  64 x 7, 600: 30.3 / 31.4;
//                    35.5 / 43.9;  4 x 10, 4000: 24.6 / 19.2; 26.9 / 24.0;  32 x 9, 4000: 78.1 /
//                    44.7; 97.4 / 73.7;  1 x 9, 16000: 32.1 / 21.6; 34.4 / 25.9
// So up to 64 rows stay with the narrow kernel where the cache is too small to repay the wide one's
// set-up; for 16-bit rows of 128 dims, where a segment's start and end take as long as three or more
// tiles of 128 positions, where sequences are short.  (Lengths are on the device: the capacity stands
// for them.)
constexpr double TN_MAX_BYTES = 4e6;
constexpr int TN_MAX_CAP = 3000;
static bool tree_short(const TreeAttnArgs& a) {
    if (a.hd > 64 && a.kv_type != KV_F32) return a.cap < TN_MAX_CAP;
    return 2.0 * a.B * a.n_kv * a.cap * a.hd * (a.kv_type == KV_F32 ? 4 : 2) < TN_MAX_BYTES;
}
static int tree_row_tile(int rows, bool short_cache) {
    if (rows <= 32) return rows <= 16 ? 16 : 32;
    return rows <= 64 && short_cache ? 64 : TW_RT;
}
static int tree_grid(int rt) { return rt == TW_RT ? tree_sms() : 2 * tree_sms(); }

size_t tree_attn_ws_bytes(int T, int n_head, int n_kv, int hd) {
    static_assert(TW_RT == 2 * 64, "half the CTAs, twice the rows: a tile of 64 rows needs as much as a wide one");
    const int rt = tree_row_tile(T * (n_head / n_kv), false);
    return 65536 + (size_t)tree_grid(rt) * 2 * tree_part_floats(rt, hd) * sizeof(float);
}

static cudaError_t tree_launch(const void* fn, dim3 grid, int threads, size_t smem, void** args, cudaStream_t st, bool pdl) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

template <int HD, int MT, int KVT>
static cudaError_t narrow_launch(const TreeAttnArgs& a, cudaStream_t st, bool pdl) {
    using F = NarrowCfg<HD, MT, KVT>;
    const void* fn = (const void*)tf_tree_attn_narrow_kernel<HD, MT, KVT>;
    static std::atomic<bool> ready[64] = {};  // set once per device; twice is harmless
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (!ready[dev]) {
        cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
        if (e != cudaSuccess) return e;
        e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return e;
        ready[dev].store(true);
    }
    TreePlan pl;
    pl.grid = tree_grid(F::RT);
    pl.rt = F::RT;
    pl.rep = a.n_head / a.n_kv;
    pl.rep_inv = (65536 + pl.rep - 1) / pl.rep;
    pl.maps = 0;
    pl.slot_rows = 0;
    TreeAttnArgs aa = a;
    void* args[] = {&aa, &pl};
    cudaError_t e = tree_launch(fn, dim3(pl.grid), TN_THREADS, F::SMEM, args, st, pdl);
    if (e != cudaSuccess) return e;
    return tree_launch((const void*)tf_tree_combine_kernel, dim3(pl.grid, F::RT / (TC_THREADS / 32)), TC_THREADS, 0, args, st, true);
}

// A 16-bit cache as a 2-D tensor map: rows of hd elements, boxes of `pt` rows x 64 elements with the
// 128-byte swizzle (one 64-dim block of an operand tile).
static bool tree_map(CUtensorMap* m, const TreeAttnArgs& a, const void* base, int pt) {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> enc{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 f = enc.load();
    if (!f) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return false;
        f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
        enc.store(f);
    }
    if (a.slot_stride % a.hd || a.hd % 64) return false;
    const long long rows = a.slot_stride / a.hd * a.n_slots;
    if (rows > 0x7FFFFFFFll) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)a.hd, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)a.hd * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)pt};
    const cuuint32_t es[2] = {1, 1};
    return f(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, int KVT>
static cudaError_t wide_launch(const TreeAttnArgs& a, cudaStream_t st, bool pdl) {
    using F = WideCfg<HD, KVT>;
    const void* fn = (const void*)tf_tree_attn_wide_kernel<HD, KVT>;
    static std::atomic<bool> ready[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (!ready[dev]) {
        cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
        if (e != cudaSuccess) return e;
        ready[dev].store(true);
    }
    TreePlan pl;
    pl.grid = tree_grid(TW_RT);
    pl.rt = TW_RT;
    pl.rep = a.n_head / a.n_kv;
    pl.rep_inv = (65536 + pl.rep - 1) / pl.rep;
    alignas(64) CUtensorMap maps[2];
    memset(maps, 0, sizeof(maps));
    pl.slot_rows = (int)(a.slot_stride / a.hd);
    pl.maps = KVT != KV_F32 && a.hd == HD && tree_map(&maps[0], a, a.kc, F::PT) && tree_map(&maps[1], a, a.vc, F::PT);
    TreeAttnArgs aa = a;
    void* args[] = {&aa, &pl, &maps[0], &maps[1]};
    cudaError_t e = tree_launch(fn, dim3(pl.grid), TW_THREADS, F::SMEM, args, st, pdl);
    if (e != cudaSuccess) return e;
    return tree_launch((const void*)tf_tree_combine_kernel, dim3(pl.grid, TW_RT / (TC_THREADS / 32)), TC_THREADS, 0, args, st, true);
}

template <int HD, int KVT>
static cudaError_t rows_launch(const TreeAttnArgs& a, cudaStream_t st, bool pdl) {
    const int rt = tree_row_tile(a.T * (a.n_head / a.n_kv), tree_short(a));
    if (rt == 16) return narrow_launch<HD, 1, KVT>(a, st, pdl);
    if (rt == 32) return narrow_launch<HD, 2, KVT>(a, st, pdl);
    if (rt == 64) return narrow_launch<HD, 4, KVT>(a, st, pdl);
    return wide_launch<HD, KVT>(a, st, pdl);
}
template <int HD>
static cudaError_t type_launch(const TreeAttnArgs& a, cudaStream_t st, bool pdl) {
    if (a.kv_type == KV_F32) return rows_launch<HD, KV_F32>(a, st, pdl);
    if (a.kv_type == KV_F16) return rows_launch<HD, KV_F16>(a, st, pdl);
    return rows_launch<HD, KV_BF16>(a, st, pdl);
}

// Tiles of 32 positions or more and a unit's cost, of units of 16 rows or more.
bool tree_attn_fits(int B, int T, int n_head, int n_kv, int cap) {
    static_assert(TN_UNIT_COST < 8 && TW_UNIT_COST < 8, "a unit's cost is within the bound");
    const long long rows = (long long)T * (n_head / n_kv);
    return (double)B * n_kv * ((rows + 15) / 16) * ((double)cap / 32 + 8) < 2147483648.0;
}

cudaError_t tree_attn_launch(const TreeAttnArgs& a, cudaStream_t st, bool pdl) {
    if (!tree_attn_fits(a.B, a.T, a.n_head, a.n_kv, a.cap)) return cudaErrorInvalidValue;
    return a.hd <= 64 ? type_launch<64>(a, st, pdl) : type_launch<128>(a, st, pdl);
}

}  // namespace tfb
