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
// exact half; a bf16 row fits one half after the scale (8 bits, and 2^-39 of the tile's maximum
// where f16 runs out of exponents).  Every tile's P V product starts from zero and joins the
// running output by an fp32 fma, so its rounding does not grow with the context.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <cstring>

#include "tree.cuh"

namespace tfb {

constexpr int TN_THREADS = 256;
constexpr int TN_TILE_BYTES = 32768;  // K and V bytes of a tile in the cache's type: 32 registers per thread
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 15.f;       // p is held as 2^15 exp(s - max): its low half keeps 2^-24 / 2^15 of it

// ---- the split of the tiles over the CTAs ---------------------------------------------------------
struct TreePlan {
    int maps;                // wide kernel, f16 cache: the tensor maps are valid
    int grid;                // CTAs of the main kernel
    int rt;                  // rows per row tile
    int pt;                  // positions per tile
    int min_tiles;           // tiles per CTA at least
};
struct TreeDesc {            // a unit split over CTAs c0..c1, found at slot c0
    int b, kvh, rtile, c1;   // b < 0: none
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
__device__ __forceinline__ int seq_tiles(const TreeSeq& s, int pt) {
    return s.n_node ? (s.n_ctx + s.n_node + pt - 1) / pt : 0;
}
__device__ __forceinline__ int seq_units(const TreeAttnArgs& a, const TreeSeq& s, int rt) {
    return a.n_kv * ((s.n_node * (a.n_head / a.n_kv) + rt - 1) / rt);
}

// This CTA's range of tiles [g0, g1): the sequence it starts in, and the global index of that
// sequence's first tile.  Block-wide; NT threads.
template <int NT>
__device__ __forceinline__ void tree_range(const TreeAttnArgs& a, const TreePlan& pl, long long& g0, long long& g1,
                                           long long& per, int& b0, long long& base0) {
    __shared__ long long wsum[NT / 32];
    __shared__ long long found_base;
    __shared__ int found_b;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int chunk = (a.B + NT - 1) / NT, lo = min(a.B, tid * chunk), hi = min(a.B, lo + chunk);
    long long mine = 0;
    for (int b = lo; b < hi; ++b) {
        const TreeSeq s = tree_seq(a, b);
        mine += (long long)seq_tiles(s, pl.pt) * seq_units(a, s, pl.rt);
        if (s.bad && blockIdx.x == 0) atomicCAS(a.err, 0, ERR_POS);
    }
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    if (tid == 0) {
        found_b = a.B;
        found_base = 0;
    }
    __syncthreads();
    long long before = inc - mine, total = 0;
    for (int w = 0; w < NT / 32; ++w) {
        if (w < warp) before += wsum[w];
        total += wsum[w];
    }
    per = (total + pl.grid - 1) / pl.grid;
    if (per < pl.min_tiles) per = pl.min_tiles;
    g0 = per * blockIdx.x;
    g1 = g0 + per < total ? g0 + per : total;
    if (g0 >= before && g0 < before + mine) {
        for (int b = lo; b < hi; ++b) {
            const TreeSeq s = tree_seq(a, b);
            const long long t = (long long)seq_tiles(s, pl.pt) * seq_units(a, s, pl.rt);
            if (g0 < before + t) {
                found_b = b;
                found_base = before;
                break;
            }
            before += t;
        }
    }
    __syncthreads();
    b0 = found_b;
    base0 = found_base;
}

// The next piece of this CTA's range [g0, g1): tiles [t0, t1) of one unit.
struct TreeSeg {
    TreeSeq s;
    int b, kvh, rtile, t0, t1, tiles, last_cta;  // last_cta: the CTA that ends the unit
};
__device__ __forceinline__ bool tree_next(const TreeAttnArgs& a, const TreePlan& pl, long long& g0, long long g1,
                                          long long per, int& b, long long& base, TreeSeg& o) {
    if (g0 >= g1) return false;
    o.s = tree_seq(a, b);
    o.tiles = seq_tiles(o.s, pl.pt);
    int units = seq_units(a, o.s, pl.rt);
    while (g0 >= base + (long long)o.tiles * units) {  // next sequence with work
        base += (long long)o.tiles * units;
        o.s = tree_seq(a, ++b);
        o.tiles = seq_tiles(o.s, pl.pt);
        units = seq_units(a, o.s, pl.rt);
    }
    const int unit = (int)((g0 - base) / o.tiles), nrt = units / a.n_kv;
    const long long u0 = base + (long long)unit * o.tiles;  // the unit's first tile
    o.b = b;
    o.kvh = unit / nrt;
    o.rtile = unit % nrt;
    o.t0 = (int)(g0 - u0);
    o.t1 = (int)(g1 - u0 < o.tiles ? g1 - u0 : o.tiles);
    o.last_cta = (int)((u0 + o.tiles - 1) / per);
    g0 = u0 + o.t1;
    return true;
}

// Rows that no unit covers (nodes from n_node on, bad sequences) are zero.
template <int NT>
__device__ __forceinline__ void tree_zero_rows(const TreeAttnArgs& a) {
    const int n4 = a.n_head * a.hd / 4, per = NT / 32;
    for (long long r = (long long)blockIdx.x * per + (threadIdx.x >> 5); r < (long long)a.B * a.T; r += (long long)gridDim.x * per) {
        const TreeSeq s = tree_seq(a, (int)(r / a.T));
        if ((int)(r % a.T) < s.n_node) continue;
        float4* o = reinterpret_cast<float4*>(a.out + r * a.ld_out);
        for (int i = threadIdx.x & 31; i < n4; i += 32) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
}

// Visibility to `node` of the 32 positions from drafted index x0 on (negative: committed
// context, always seen); nothing from n_node on.
__device__ __forceinline__ uint32_t tree_window(const TreeAttnArgs& a, const TreeSeq& s, int b, int node, int x0) {
    auto word = [&](int w) -> unsigned long long {  // nodes 64 w .. 64 w + 63
        if (w < 0) return ~0ull;
        if (64 * w >= s.n_node || node >= s.n_node) return 0ull;
        unsigned long long v;
        if (a.mask) v = a.mask[((size_t)b * a.T + node) * ((a.T + 63) / 64) + w];
        else v = 64 * w > node ? 0ull : (node - 64 * w >= 63 ? ~0ull : (2ull << (node - 64 * w)) - 1);
        const int left = s.n_node - 64 * w;
        return left >= 64 ? v : v & ((1ull << left) - 1);
    };
    if (x0 <= -32) return 0xFFFFFFFFu;
    const int w = x0 >> 6, sh = x0 & 63;
    const unsigned long long lo = word(w) >> sh;
    return (uint32_t)(sh > 32 ? lo | (word(w + 1) << (64 - sh)) : lo);
}

// ---- small pieces ---------------------------------------------------------------------------------
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e for -126 <= e <= 127
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
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
// two values into their high halves (packed) and what the halves leave
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = pack_half2(x, y);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    lo = pack_half2(x - f.x, y - f.y);
}
// the same by truncation: the high half keeps 10 bits behind the first (exact in f16 from 2^-14
// on), the low half the rest
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
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- narrow trees: mma.sync, up to 64 rows per row tile ----------------------------------------------
// One CTA of 8 warps per range of tiles, two CTAs per SM.  A tile is 32 KB of cache (K and V),
// copied into shared memory by cp.async one tile ahead while the current one is computed; fp32
// and bf16 tiles are then split into f16 halves in a second buffer, each thread taking the
// vectors that it copied itself (no barrier in between), f16 tiles alternate between the two
// buffers.  Operand rows are HD halves, 16-byte chunk c of row r at c ^ (r & 7).
// Warp (m, g): 16 rows of row block m, the positions of group g of the tile; each keeps its own
// running maximum, sum and output, and the groups meet through shared memory when a unit ends.
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
__global__ void __launch_bounds__(TN_THREADS, 2) tf_tree_attn_narrow_kernel(const TreeAttnArgs a, const TreePlan pl) {
    using F = NarrowCfg<HD, MT, KVT>;
    constexpr int PT = F::PT, RT = F::RT, NG = F::NG, PB = F::PB, NLO = F::NLO, ESZ = F::ESZ;
    constexpr int VEC = 16 / ESZ, VPR = HD / VEC, NV = TN_TILE_BYTES / 2 / 16 / TN_THREADS;  // vectors: elements, per row, per thread
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ float qscale[RT];
    __shared__ unsigned tmax[4];        // maxima of K, V (bits) of this tile and the next
    __shared__ unsigned badrow[TREE_MAX_NODES / 32];  // drafted rows of the unit with non-finite values
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rep = a.n_head / a.n_kv, hd = a.hd;
    const uint32_t sb = smem_u32(smem);
    const uint32_t qh = sb + 2 * TN_TILE_BYTES, ql = qh + F::Q_BYTES;
    const int rep_inv = (65536 + rep - 1) / rep;  // row / rep for rows < 2048 and rep <= 8
    auto div_rep = [&](int x) { return (x * rep_inv) >> 16; };
    const int wm = warp % MT, wg = warp / MT;  // row block, position group
    const bool active = wg < NG;
    const int g8 = lane >> 2, q4 = lane & 3;

    pdl_trigger();
    pdl_wait();
    TreeDesc* desc = static_cast<TreeDesc*>(a.ws);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + 65536);
    long long g0, g1, per, base;
    int b;
    tree_range<TN_THREADS>(a, pl, g0, g1, per, b, base);
    if (tid == 0) desc[blockIdx.x].b = -1;

    TreeSeg sg;
    while (tree_next(a, pl, g0, g1, per, b, base, sg)) {
        const TreeSeq s = sg.s;
        const int kvh = sg.kvh, rtile = sg.rtile, t0 = sg.t0, t1 = sg.t1;
        const int end = s.n_ctx + s.n_node, rows = s.n_node * rep;
        const size_t off = (size_t)s.slot * a.slot_stride + (size_t)kvh * a.cap * hd;
        const uint8_t* kp = static_cast<const uint8_t*>(a.kc) + off * ESZ;
        const uint8_t* vp = static_cast<const uint8_t*>(a.vc) + off * ESZ;

        // tile t into its buffer: vector v = tid + i * threads of the PT x HD tile, K then V
        // (f16: at its operand place, the buffers alternating; else in the order of the threads)
        auto place = [&](int t, int i) -> uint32_t {
            const int v = tid + i * TN_THREADS, r = v / VPR, c = v % VPR;
            if (KVT != KV_F16) return sb + 16u * v;
            return sb + (uint32_t)(t & 1) * TN_TILE_BYTES + (uint32_t)r * (HD * 2) + (((uint32_t)c ^ (r & 7)) << 4);
        };
        auto load = [&](int t) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int v = tid + i * TN_THREADS, p = t * PT + v / VPR, c = (v % VPR) * VEC;
                const bool in = p < end && c < hd;
                const size_t e = in ? ((size_t)p * hd + c) * ESZ : 0;
                const uint32_t o = place(t, i);
                cp_async16(o, kp + e, in);
                cp_async16(o + TN_TILE_BYTES / 2, vp + e, in);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        load(t0);
        // the rows' queries, TPR threads per row: scaled to [2^14, 2^15), two halves
        {
            constexpr int TPR = TN_THREADS / RT < HD / 8 ? TN_THREADS / RT : HD / 8, UPT = HD / 8 / TPR;  // 8-dim units per thread
            const int r = tid / TPR, rr = rtile * RT + r, j0 = tid % TPR;
            if (r < RT) {
                float x[UPT][8];
                uint32_t mb = 0;
                const int node = div_rep(rr);
                const float* qp = a.q + ((size_t)b * a.T + node) * a.ld_q + (size_t)(kvh * rep + rr - node * rep) * hd;
#pragma unroll
                for (int i = 0; i < UPT; ++i) {
                    const int d = (j0 + i * TPR) * 8;
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f), z = y;
                    if (rr < rows && d < hd) {
                        y = *reinterpret_cast<const float4*>(qp + d);
                        z = *reinterpret_cast<const float4*>(qp + d + 4);
                    }
                    x[i][0] = y.x, x[i][1] = y.y, x[i][2] = y.z, x[i][3] = y.w;
                    x[i][4] = z.x, x[i][5] = z.y, x[i][6] = z.z, x[i][7] = z.w;
                }
#pragma unroll
                for (int i = 0; i < UPT; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) mb = max(mb, finite_abs_bits(x[i][j]));
#pragma unroll
                for (int o = 1; o < TPR; o <<= 1) mb = max(mb, __shfl_xor_sync(0xFFFFFFFFu, mb, o));
                const int e = half_exponent(mb);
                const float sc = pow2i(-e);
#pragma unroll
                for (int i = 0; i < UPT; ++i) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) split2(x[i][2 * j] * sc, x[i][2 * j + 1] * sc, hi[j], lo[j]);
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
        __syncthreads();

        float O[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) O[i][0] = O[i][1] = O[i][2] = O[i][3] = 0.f;

        for (int t = t0; t < t1; ++t) {
            int ek = 0, ev = 0;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            // non-finite values of drafted rows leave the V tile (another row's zero weight
            // must not meet them); rows that see them take them up at the end
            const bool tail = (t + 1) * PT > s.n_ctx;
            uint32_t kh = sb + (KVT == KV_F16 ? (uint32_t)(t & 1) * TN_TILE_BYTES : TN_TILE_BYTES), vh = kh + TN_TILE_BYTES / 2;
            uint32_t mk = 0, mv = 0;
            if (KVT != KV_F16 || tail) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const uint32_t o = place(t, i) + TN_TILE_BYTES / 2;
                    uint4 x = ld_shared16(o);
                    const int p = t * PT + (tid + i * TN_THREADS) / VPR;
                    if (tail && p >= s.n_ctx && zero_nonfinite<KVT>(x)) {
                        atomicOr(&badrow[(p - s.n_ctx) >> 5], 1u << ((p - s.n_ctx) & 31));
                        st_shared16(o, {x.x, x.y, x.z, x.w});
                    }
                    if (KVT != KV_F16) {
                        mv = max(mv, max_bits<KVT>(x));
                        mk = max(mk, max_bits<KVT>(ld_shared16(o - TN_TILE_BYTES / 2)));
                    }
                }
            }
            if (KVT != KV_F16) {
                mk = __reduce_max_sync(0xFFFFFFFFu, mk);
                mv = __reduce_max_sync(0xFFFFFFFFu, mv);
                if (lane == 0) {
                    atomicMax(&tmax[2 * (t & 1)], mk);
                    atomicMax(&tmax[2 * (t & 1) + 1], mv);
                }
                __syncthreads();  // the maxima; the last tile's operands are free
                ek = half_exponent(tmax[2 * (t & 1)]);
                ev = half_exponent(tmax[2 * (t & 1) + 1]);
                if (tid < 2) tmax[2 * (~t & 1) + tid] = 0;  // the next tile's, last read a barrier ago
                const float sk = pow2i(-ek), sv = pow2i(-ev);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int v = tid + i * TN_THREADS, r = v / VPR, c = v % VPR;
#pragma unroll
                    for (int which = 0; which < 2; ++which) {
                        const uint4 x = ld_shared16(place(t, i) + which * (TN_TILE_BYTES / 2));
                        const float f = which ? sv : sk;
                        const uint32_t dst = which ? vh : kh;
                        if (KVT == KV_F32) {
                            uint32_t h0, l0, h1, l1;
                            split2(__uint_as_float(x.x) * f, __uint_as_float(x.y) * f, h0, l0);
                            split2(__uint_as_float(x.z) * f, __uint_as_float(x.w) * f, h1, l1);
                            const uint32_t o = dst + (uint32_t)r * (HD * 2) + ((((uint32_t)c >> 1) ^ (r & 7)) << 4) + (c & 1) * 8;
                            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(o), "r"(h0), "r"(h1) : "memory");
                            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(o + F::TILE_H), "r"(l0), "r"(l1) : "memory");
                        } else {
                            uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                w[j] = pack_half2(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xFFFF0000u) * f);
                            st_shared16(dst + (uint32_t)r * (HD * 2) + (((uint32_t)c ^ (r & 7)) << 4), w);
                        }
                    }
                }
            }
            __syncthreads();
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
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    uint32_t ah[4], al[4];
                    {
                        const int r = wm * 16 + (lane & 15), c = 2 * kk + (lane >> 4);
                        const uint32_t o = (uint32_t)r * (HD * 2) + (((uint32_t)c ^ (r & 7)) << 4);
                        ldsm4(ah, qh + o);
                        ldsm4(al, ql + o);
                    }
#pragma unroll
                    for (int nb = 0; nb < PB / 16; ++nb) {
                        const int r = pl0 + nb * 16 + (lane & 7) + ((lane >> 4) << 3), c = 2 * kk + ((lane >> 3) & 1);
                        const uint32_t o = kh + (uint32_t)r * (HD * 2) + (((uint32_t)c ^ (r & 7)) << 4);
                        uint32_t bh[4];
                        ldsm4(bh, o);
                        mma16816(S[2 * nb], ah, bh[0], bh[1]);
                        mma16816(S[2 * nb + 1], ah, bh[2], bh[3]);
                        mma16816(S1[2 * nb], al, bh[0], bh[1]);
                        mma16816(S1[2 * nb + 1], al, bh[2], bh[3]);
                        if (NLO == 2) {
                            uint32_t bl[4];
                            ldsm4(bl, o + F::TILE_H);
                            mma16816(S1[2 * nb], ah, bl[0], bl[1]);
                            mma16816(S1[2 * nb + 1], ah, bl[2], bl[3]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < PB / 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) S[i][j] += S1[i][j];
                // base-2 scores, masks, running maximum and sum of this thread's two rows
                float alpha[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int r = wm * 16 + g8 + 8 * half;
                    const float f = qscale[r] * fk;
                    float mx = m[half];
                    if (!tail) {
#pragma unroll
                        for (int i = 0; i < PB / 8; ++i)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                S[i][2 * half + j] *= f;
                                mx = fmaxf(mx, S[i][2 * half + j]);
                            }
                    } else {
                        // bit i of vis: position i of the step is seen
                        const int node = div_rep(rtile * RT + r), x0 = t * PT + pl0 - s.n_ctx;
                        const uint32_t vis = tree_window(a, s, b, node, x0);
#pragma unroll
                        for (int i = 0; i < PB / 8; ++i)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                S[i][2 * half + j] = (vis >> (i * 8 + 2 * q4 + j)) & 1 ? S[i][2 * half + j] * f : -INFINITY;
                                mx = fmaxf(mx, S[i][2 * half + j]);
                            }
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
                for (int i = 0; i < PB / 16; ++i) {
                    split2(S[2 * i][0], S[2 * i][1], ph[i][0], pq[i][0]);
                    split2(S[2 * i][2], S[2 * i][3], ph[i][1], pq[i][1]);
                    split2(S[2 * i + 1][0], S[2 * i + 1][1], ph[i][2], pq[i][2]);
                    split2(S[2 * i + 1][2], S[2 * i + 1][3], ph[i][3], pq[i][3]);
                }
#pragma unroll
                for (int db = 0; db < HD / 16; ++db) {
                    float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < PB / 16; ++i) {
                        const int r = pl0 + i * 16 + (lane & 15), c = 2 * db + (lane >> 4);
                        const uint32_t o = vh + (uint32_t)r * (HD * 2) + (((uint32_t)c ^ (r & 7)) << 4);
                        uint32_t bh[4];
                        ldsm4t(bh, o);
                        mma16816(d0, ph[i], bh[0], bh[1]);
                        mma16816(d1, ph[i], bh[2], bh[3]);
                        mma16816(d0, pq[i], bh[0], bh[1]);
                        mma16816(d1, pq[i], bh[2], bh[3]);
                        if (NLO == 2) {
                            uint32_t bl[4];
                            ldsm4t(bl, o + F::TILE_H);
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
        for (int i = tid; i < RT * (HD / 4); i += TN_THREADS) {
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4, rr = rtile * RT + r;
            if (rr >= rows || d >= hd) continue;
            float M = -INFINITY;
#pragma unroll
            for (int g = 0; g < NG; ++g) M = fmaxf(M, fin[((size_t)g * RT + r) * (HD + 4) + HD]);
            const float ref = M == -INFINITY ? 0.f : M;
            float L = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float* fr = fin + ((size_t)g * RT + r) * (HD + 4);
                const float w = exp2_fast(fr[HD] - ref);
                const float4 x = *reinterpret_cast<const float4*>(fr + d);
                L = fmaf(fr[HD + 1], w, L);
                o.x = fmaf(x.x, w, o.x);
                o.y = fmaf(x.y, w, o.y);
                o.z = fmaf(x.z, w, o.z);
                o.w = fmaf(x.w, w, o.w);
            }
            const int node = div_rep(rr);
            for (int w = 0; w < TREE_MAX_NODES / 32 && anybad; ++w)  // non-finite drafted values that the row sees
                for (unsigned bits = badrow[w]; bits; bits &= bits - 1) {
                    const int x = w * 32 + __ffs(bits) - 1;
                    const bool vis = a.mask ? (a.mask[((size_t)b * a.T + node) * ((a.T + 63) / 64) + (x >> 6)] >> (x & 63)) & 1 : x <= node;
                    if (!vis) continue;
                    float* oo = &o.x;
                    for (int j = 0; j < 4; ++j) {
                        const float v = kv_load(a.vc, (long long)off + (long long)(s.n_ctx + x) * hd + d + j, KVT);
                        if (!(fabsf(v) < INFINITY)) oo[j] += v;
                    }
                }
            if (whole) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                o.x = L == 0.f ? 0.f : o.x * inv;
                o.y = L == 0.f ? 0.f : o.y * inv;
                o.z = L == 0.f ? 0.f : o.z * inv;
                o.w = L == 0.f ? 0.f : o.w * inv;
                *reinterpret_cast<float4*>(a.out + ((size_t)b * a.T + node) * a.ld_out + (size_t)(kvh * rep + rr - node * rep) * hd + d) = o;
            } else {
                *reinterpret_cast<float4*>(part + (size_t)r * hd + d) = o;
                if (d == 0) {
                    part[(size_t)RT * hd + r] = M;
                    part[(size_t)RT * hd + RT + r] = L;
                }
            }
        }
        if (!whole && t0 == 0 && tid == 0)
            desc[blockIdx.x] = TreeDesc{b, kvh, rtile, sg.last_cta};
        __syncthreads();
    }
    tree_zero_rows<TN_THREADS>(a);
}

// ---- wide trees: tcgen05, 128 rows per row tile -------------------------------------------------------
// One CTA per SM and range of tiles, four warpgroups:
//   0, 1  softmax streams: even and odd tiles of a segment, a thread per row with a running
//         maximum, sum and output of its own (registers); no shuffles, no exchange until the end;
//   2     loaders: a tile's K and V rows arrive by one 1-D bulk copy each, are split into f16
//         halves and written as MMA operands (rows of 64 dims, 128-byte swizzle);
//   3     MMA issue (one thread).
// Tensor memory: S_0, S_1 (PT columns each) and D_0, D_1 (HD columns each).  QK: S_w = Q K^T,
// Q from shared memory, the tile K-major.  The softmax thread overwrites its scores in place,
// CH columns at a time, with the high halves of p (CH / 2 columns) and the low ones, the A
// operand of PV: D_w = P V, the same tile layout read MN-major; D_w starts from zero for every
// tile and joins the registers' output.  QK of tile i + 1 is issued before PV of tile i, so the
// tensor pipe works while a stream is in its softmax.
constexpr int TW_THREADS = 512;
constexpr int TW_RT = 128;

constexpr int TW_LOADERS = 6;  // loader warps: warpgroup 2 and the last two warps of warpgroup 3

template <int HD, int KVT>
struct WideCfg {
    static constexpr int ESZ = KVT == KV_F32 ? 4 : 2;
    static constexpr int PT = KVT == KV_F32 && HD == 128 ? 64 : 128;
    static constexpr int NLO = KVT == KV_F32 ? 2 : 1;
    static constexpr int HALF = PT * HD * 2;              // bytes of one half of a K or V tile
    static constexpr int RAW = PT * HD * ESZ;             // bytes of a raw K or V tile
    // operand stages, and raw buffers of one K or V tile each
    static constexpr int OS = KVT == KV_F16 ? (HD == 64 ? 4 : 2) : (KVT == KV_BF16 && HD == 64 ? 2 : 1);
    static constexpr int RS = HD == 64 ? (KVT == KV_F32 ? 3 : 4) : 2;
    static constexpr int QH = TW_RT * HD * 2;             // bytes of one half of Q
    static constexpr int Q_OFF = 0;
    static constexpr int K_OFF = 2 * QH;
    static constexpr int V_OFF = K_OFF + OS * NLO * HALF;
    static constexpr int RAW_OFF = V_OFF + OS * NLO * HALF;
    static constexpr int SMEM = RAW_OFF + (KVT == KV_F16 ? 0 : RS * RAW) + 1024;
    // registers per thread of the softmax warpgroups and of the other two (512 in all, four
    // warpgroups of 128 at launch)
    static constexpr int REG_S = HD == 64 ? 168 : 184, REG_L = HD == 64 ? 88 : 72;
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
    uint64_t rawfull[4], rawfree[4];              // raw tiles
    uint64_t kfull[4], kfree[4], vfull[4], vfree[4];  // operand stages
    uint64_t sfull[2], pfull[2], dfull[2], qfull, done;
    uint32_t tmem;
    int abort;
    unsigned tmax[4];
    int ek[4], ev[4];                             // scale exponents of the last four tiles
    unsigned badrow[8][TREE_MAX_NODES / 32];      // drafted rows with non-finite values, by segment
    float qscale[TW_RT];
    float2 ml[2][TW_RT];                          // the streams' row maxima and sums
};

// Exponent that puts a tile's maximum at 2^8: room for 2^7 more before f16 overflows, and 2^8
// less before the low halves run out of exponents.
__device__ __forceinline__ int tile_exponent(uint32_t maxbits) {
    const int e = (int)(maxbits >> 23) - 127 - 8;
    return e < -126 ? -126 : (e > 126 ? 126 : e);
}

template <int HD, int KVT>
__global__ void __launch_bounds__(TW_THREADS, 1) tf_tree_attn_wide_kernel(const TreeAttnArgs a, const TreePlan pl,
                                                                           const __grid_constant__ CUtensorMap kmap,
                                                                           const __grid_constant__ CUtensorMap vmap) {
    using F = WideCfg<HD, KVT>;
    constexpr int PT = F::PT, NLO = F::NLO, ESZ = F::ESZ, OS = F::OS, RS = F::RS, CH = F::CH;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(16) WideShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
    const int rep = a.n_head / a.n_kv, hd = a.hd;
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    volatile int* abort_flag = &sh.abort;
    const int rep_inv = (65536 + rep - 1) / rep;  // row / rep for rows < 2048 and rep <= 8

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    if (tid == 32) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(&sh.rawfull[i], 1);
            mbar_init(&sh.rawfree[i], TW_LOADERS);
            mbar_init(&sh.kfull[i], TW_LOADERS);
            mbar_init(&sh.vfull[i], TW_LOADERS);
            mbar_init(&sh.kfree[i], 1);
            mbar_init(&sh.vfree[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.sfull[i], 1);
            mbar_init(&sh.pfull[i], 128);
            mbar_init(&sh.dfull[i], 1);
        }
        mbar_init(&sh.qfull, 256);
        mbar_init(&sh.done, 1);
        sh.abort = 0;
        for (int i = 0; i < 4; ++i) sh.tmax[i] = 0;
        mbar_fence_init();
    }
    pdl_trigger();
    pdl_wait();
    TreeDesc* desc = static_cast<TreeDesc*>(a.ws);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + 65536);
    if (tid == 0) desc[blockIdx.x].b = -1;
    long long g0, g1, per, base;
    int b;
    tc_fence_before();
    tree_range<TW_THREADS>(a, pl, g0, g1, per, b, base);  // (block barriers inside)
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    TreeSeg sg;

    // Every role walks the same segments and tiles; after an abort the waits return at once and
    // the roles run on without effect, so that all of them meet at every barrier.
    // A tile that needs no work on its values (f16, all of it committed context) goes straight
    // to its operand stage through the tensor maps.
    auto direct = [&](const TreeSeg& g, int t) { return KVT == KV_F16 && pl.maps && (t + 1) * PT <= g.s.n_ctx; };
    if (wg >= 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::REG_L));
    if (wg == 2 || warp >= 14) {
        constexpr int LT = TW_LOADERS * 32;
        const int lt = wg == 2 ? tid - 256 : tid - 320;
        int n = 0, nr = 0, seg = 0;  // running tile, raw buffer and segment
        int e2k = 0, e2v = 0;        // current exponents of K and V
        while (tree_next(a, pl, g0, g1, per, b, base, sg)) {
            const TreeSeq s = sg.s;
            const int end = s.n_ctx + s.n_node;
            if (lt < TREE_MAX_NODES / 32) sh.badrow[seg & 7][lt] = 0;  // read by others long ago
            named_bar<2, LT>();
            for (int t = sg.t0; t < sg.t1; ++t, ++n) {
                const int os = n % OS, rows = min(PT, end - t * PT);
#pragma unroll 1
                for (int which = 0; which < 2; ++which) {
                    uint64_t* full = which ? &sh.vfull[os] : &sh.kfull[os];
                    uint64_t* free = which ? &sh.vfree[os] : &sh.kfree[os];
                    const uint32_t off = (which ? F::V_OFF : F::K_OFF) + os * NLO * F::HALF;
                    // the operand stage is free once the MMAs of OS tiles ago are done
                    if (direct(sg, t)) {
                        if (lane == 0) {
                            if (n >= OS) mbar_wait(free, (n / OS - 1) & 1, a.err, ERR_WAIT_EMPTY, abort_flag);
                            if (lt == 0 && !*abort_flag) {
                                mbar_expect_tx(full, F::HALF);
                                const int row = (int)(((size_t)s.slot * a.slot_stride) / hd + (size_t)sg.kvh * a.cap) + t * PT;
#pragma unroll
                                for (int c = 0; c < HD / 64; ++c)
                                    asm volatile(
                                        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                                        "[%1, {%2, %3}], [%4];" ::"r"(sb + off + c * PT * 128),
                                        "l"(reinterpret_cast<uint64_t>(which ? &vmap : &kmap)), "r"(64 * c), "r"(row), "r"(smem_u32(full))
                                        : "memory");
                            } else {
                                mbar_arrive(full);
                            }
                        }
                        continue;
                    }
                    const int rs = nr % RS;
                    uint8_t* raw = smem + F::RAW_OFF + rs * F::RAW;
                    if (KVT != KV_F16) mbar_wait(&sh.rawfull[rs], (nr / RS) & 1, a.err, ERR_WAIT_FULL, abort_flag);
                    if (n >= OS) mbar_wait(free, (n / OS - 1) & 1, a.err, ERR_WAIT_EMPTY, abort_flag);
                    __syncwarp();
                    ++nr;
                    constexpr int UNITS = PT * HD / 8, UPR = HD / 8;  // 8-element units, per row
                    if (KVT != KV_F16 && which && (t + 1) * PT > s.n_ctx)  // non-finite drafted values leave the operand (see the narrow kernel)
                        for (int v = lt; v < UNITS; v += LT) {
                            const int r = v / UPR, c = (v % UPR) * 8, p = t * PT + r;
                            if (r >= rows || c >= hd || p < s.n_ctx) continue;
                            uint4* x = reinterpret_cast<uint4*>(raw + ((size_t)r * hd + c) * ESZ);
                            for (int k = 0; k < ESZ / 2; ++k) {
                                uint4 y = x[k];
                                if (zero_nonfinite<KVT>(y)) {
                                    x[k] = y;
                                    atomicOr(&sh.badrow[seg & 7][(p - s.n_ctx) >> 5], 1u << ((p - s.n_ctx) & 31));
                                }
                            }
                        }
                    const uint32_t dst = sb + off, rawa = smem_u32(raw);
                    // converted with the last tile's exponent; when the tile's maximum turns out not
                    // to fit it (seldom), once more with its own
                    for (;;) {
                        const int ec = which ? e2v : e2k;
                        const float f = pow2i(-ec);
                        float mf = 0.f;       // largest |x| of fp32 values
                        uint32_t mw = 0;      // largest |x| of bf16 values, two lanes
#pragma unroll 4
                        for (int v = lt; v < UNITS; v += LT) {
                            const int r = v / UPR, c = v % UPR;
                            uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
                            if (r < rows && c * 8 < hd) {
                                const uint32_t x = rawa + (uint32_t)((r * hd + c * 8) * ESZ);
                                if (KVT == KV_F16) {  // the few such tiles come straight from the cache
                                    const int p = t * PT + r;
                                    const size_t at = (size_t)s.slot * a.slot_stride + ((size_t)sg.kvh * a.cap + p) * hd + c * 8;
                                    x0 = *reinterpret_cast<const uint4*>(static_cast<const __half*>(which ? a.vc : a.kc) + at);
                                    if (which && p >= s.n_ctx && zero_nonfinite<KVT>(x0))
                                        atomicOr(&sh.badrow[seg & 7][(p - s.n_ctx) >> 5], 1u << ((p - s.n_ctx) & 31));
                                } else {
                                    x0 = ld_shared16(x);
                                    if (KVT == KV_F32) x1 = ld_shared16(x + 16);
                                }
                            }
                            const uint32_t o = dst + wide_off(PT, r, c);
                            if (KVT == KV_F32) {
                                uint32_t hi[4], lo[4];
                                const uint32_t w[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const float2 y = make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
                                    mf = fmaxf(mf, fmaxf(fabsf(y.x), fabsf(y.y)));
                                    split2t(__fmul2_rn(y, make_float2(f, f)), hi[j], lo[j]);
                                }
                                st_shared16(o, hi);
                                st_shared16(o + F::HALF, lo);
                            } else {
                                uint32_t w[4] = {x0.x, x0.y, x0.z, x0.w};
                                if (KVT == KV_BF16) {
#pragma unroll
                                    for (int j = 0; j < 4; ++j) {
                                        mw = __vmaxu2(mw, w[j] & 0x7FFF7FFFu);
                                        w[j] = pack_half2(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xFFFF0000u) * f);
                                    }
                                }
                                st_shared16(o, w);
                            }
                        }
                        uint32_t mb = KVT == KV_F32 ? __float_as_uint(mf) : max(mw << 16, mw & 0xFFFF0000u);
                        if (KVT != KV_F16 && __any_sync(0xFFFFFFFFu, mb >= 0x7F800000u)) {  // infinities or NaN: the finite maximum
                            mb = 0;
                            for (int v = lt; v < UNITS; v += LT) {
                                const int r = v / UPR, c = v % UPR;
                                if (r >= rows || c * 8 >= hd) continue;
                                const uint32_t x = rawa + (uint32_t)((r * hd + c * 8) * ESZ);
                                mb = max(mb, max_bits<KVT>(ld_shared16(x)));
                                if (KVT == KV_F32) mb = max(mb, max_bits<KVT>(ld_shared16(x + 16)));
                            }
                            __syncwarp();
                        }
                        if (KVT == KV_F16) break;
                        mb = __reduce_max_sync(0xFFFFFFFFu, mb);
                        unsigned* tm = &sh.tmax[2 * (n & 1) + which];
                        if (lane == 0) atomicMax(tm, mb);
                        named_bar<2, LT>();
                        const uint32_t all = *tm;
                        // fits: the maximum is within [2^0, 2^15) after the scale
                        const int e = tile_exponent(all), d = e - ec;
                        if (all == 0 || d == 0 || (d > -8 && d < 7)) break;
                        named_bar<2, LT>();  // every thread has read the exponent's base
                        if (which) e2v = e;
                        else e2k = e;
                    }
                    if (lt == 0) {
                        sh.tmax[2 * (~n & 1) + which] = 0;  // the next tile's, read last a tile ago
                        (which ? sh.ev : sh.ek)[n & 3] = which ? e2v : e2k;
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(full);
                        if (KVT != KV_F16) mbar_arrive(&sh.rawfree[rs]);
                    }
                }
            }
            ++seg;
        }
        // after an abort: copies of the last stages may still be on their way
        if (lt == 0 && *abort_flag)
            for (int i = max(0, n - OS); i < n; ++i) {
                mbar_wait(&sh.kfull[i % OS], (i / OS) & 1, a.err, ERR_WAIT_FULL, nullptr);
                mbar_wait(&sh.vfull[i % OS], (i / OS) & 1, a.err, ERR_WAIT_FULL, nullptr);
            }
    } else if (warp == 13) {
        // raw copies, RS buffers ahead
        if (KVT != KV_F16 && lane == 0) {
            int nr = 0, last[RS];  // last copy into each buffer
#pragma unroll
            for (int i = 0; i < RS; ++i) last[i] = -1;
            while (tree_next(a, pl, g0, g1, per, b, base, sg))
                for (int t = sg.t0; t < sg.t1; ++t) {
                    const int rows = min(PT, sg.s.n_ctx + sg.s.n_node - t * PT);
                    const uint32_t bytes = (uint32_t)(rows * hd * ESZ);
                    const size_t off = ((size_t)sg.s.slot * a.slot_stride + ((size_t)sg.kvh * a.cap + (size_t)t * PT) * hd) * ESZ;
                    for (int which = 0; which < 2; ++which, ++nr) {
                        const int rs = nr % RS;
                        if (nr >= RS) mbar_wait(&sh.rawfree[rs], (nr / RS - 1) & 1, a.err, ERR_WAIT_EMPTY, abort_flag);
                        if (*abort_flag) continue;
                        mbar_expect_tx(&sh.rawfull[rs], bytes);
                        bulk_g2s(smem + F::RAW_OFF + rs * F::RAW, static_cast<const uint8_t*>(which ? a.vc : a.kc) + off, bytes, &sh.rawfull[rs]);
                        last[rs] = nr / RS;
                    }
                }
            if (*abort_flag)  // copies that may still be on their way
                for (int i = 0; i < RS; ++i)
                    if (last[i] >= 0) mbar_wait(&sh.rawfull[i], last[i] & 1, a.err, ERR_WAIT_FULL, nullptr);
        }
        __syncwarp();
    } else if (warp == 12) {
        // D f32, A / B f16, M = 128: QK with N = PT, both K-major; PV with N = HD, B MN-major
        constexpr uint32_t iqk = (1u << 4) | ((uint32_t)(PT >> 3) << 17) | ((uint32_t)(TW_RT >> 4) << 24);
        constexpr uint32_t ipv = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(TW_RT >> 4) << 24);
        const uint32_t lead = elect_lane(), tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        int n = 0, seg = 0;
        int cnt0 = 0, cnt1 = 0;  // PVs issued per stream
        bool ok = true;
        auto wait = [&](uint64_t* bar, int parity) {
            ok = __all_sync(0xFFFFFFFFu, ok && mbar_wait(bar, parity & 1, a.err, ERR_WAIT_FULL, abort_flag));
        };
        auto pv = [&](int m, int w) {  // tile m of the run, stream w
            const int os = m % OS;
            wait(&sh.pfull[w], w ? cnt1 : cnt0);
            wait(&sh.vfull[os], m / OS);
            if (w) ++cnt1;
            else ++cnt0;
            if (!ok) return;
            tc_fence_after();
            const uint32_t d = tm + 256 + w * HD, p = tm + w * 128;
            const uint64_t vh = wide_desc(sb + F::V_OFF + os * NLO * F::HALF, PT * 128);
            const uint64_t vl = wide_desc(sb + F::V_OFF + os * NLO * F::HALF + (NLO - 1) * F::HALF, PT * 128);
#pragma unroll
            for (int j = 0; j < PT / 16; ++j) {  // 16 positions: 2048 bytes of rows; p's halves in blocks of CH columns
                const uint32_t ph = CH == 32 ? p + 32 * (j / 2) + 8 * (j % 2) : p + 16 * j;
                wide_mma_ts(d, ph, vh + 128u * j, ipv, j > 0, lead);
                wide_mma_ts(d, ph + CH / 2, vh + 128u * j, ipv, 1, lead);
                if (NLO == 2) wide_mma_ts(d, ph, vl + 128u * j, ipv, 1, lead);
            }
            wide_commit(&sh.vfree[os], lead);
            wide_commit(&sh.dfull[w], lead);
        };
        while (tree_next(a, pl, g0, g1, per, b, base, sg)) {
            wait(&sh.qfull, seg);
            for (int t = sg.t0; t < sg.t1; ++t, ++n) {
                const int w = (t - sg.t0) & 1, os = n % OS;
                wait(&sh.kfull[os], n / OS);
                if (ok) {
                    tc_fence_after();
                    const uint32_t d = tm + w * 128;
                    const uint64_t kb = wide_desc(sb + F::K_OFF + os * NLO * F::HALF, 16), qb = wide_desc(sb + F::Q_OFF, 16);
#pragma unroll
                    for (int j = 0; j < HD / 16; ++j) {  // 16 dims: 32 bytes along the rows of a 64-dim block
                        const uint64_t q = qb + ((j / 4) * (TW_RT * 128) + (j % 4) * 32) / 16;
                        const uint64_t k = kb + ((j / 4) * (PT * 128) + (j % 4) * 32) / 16;
                        wide_mma_ss(d, q, k, iqk, j > 0, lead);
                        wide_mma_ss(d, q + F::QH / 16, k, iqk, 1, lead);
                        if (NLO == 2) wide_mma_ss(d, q, k + F::HALF / 16, iqk, 1, lead);
                    }
                    wide_commit(&sh.kfree[os], lead);
                    wide_commit(&sh.sfull[w], lead);
                }
                if (t > sg.t0) pv(n - 1, w ^ 1);
            }
            pv(n - 1, (sg.t1 - 1 - sg.t0) & 1);
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
        while (tree_next(a, pl, g0, g1, per, b, base, sg)) {
            const TreeSeq s = sg.s;
            const int rows = s.n_node * rep;
            {   // queries, HD / 8 lanes per row: scaled to [2^14, 2^15), two halves
                constexpr int LPR = HD / 8, RPW = 32 / LPR, STEPS = TW_RT / (8 * RPW);
                float4 x[STEPS][2];
                const int c = lane % LPR;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const int r = (i * 8 + warp) * RPW + lane / LPR, q = sg.rtile * TW_RT + r, nd = (q * rep_inv) >> 16;
                    const float* qp = a.q + ((size_t)sg.b * a.T + nd) * a.ld_q + (size_t)(sg.kvh * rep + q - nd * rep) * hd + c * 8;
                    x[i][0] = x[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (q < rows && c * 8 < hd) {
                        x[i][0] = reinterpret_cast<const float4*>(qp)[0];
                        x[i][1] = reinterpret_cast<const float4*>(qp)[1];
                    }
                }
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const int r = (i * 8 + warp) * RPW + lane / LPR;
                    const float y[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w, x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
                    uint32_t mb = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) mb = max(mb, finite_abs_bits(y[j]));
#pragma unroll
                    for (int o = 1; o < LPR; o <<= 1) mb = max(mb, __shfl_xor_sync(0xFFFFFFFFu, mb, o));
                    const int e = half_exponent(mb);
                    const float sc = pow2i(-e);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) split2(y[2 * j] * sc, y[2 * j + 1] * sc, hi[j], lo[j]);
                    const uint32_t o = sb + F::Q_OFF + wide_off(TW_RT, r, c);
                    st_shared16(o, hi);
                    st_shared16(o + F::QH, lo);
                    if (c == 0) sh.qscale[r] = pow2i(e) * (kLog2e / sqrtf((float)hd));
                }
                fence_async();
                mbar_arrive(&sh.qfull);
                named_bar<1, 256>();
            }
            const float qs = sh.qscale[row];
            const int rr = sg.rtile * TW_RT + row, node = (rr * rep_inv) >> 16;
            float O[HD], m = -INFINITY, l = 0.f;
#pragma unroll
            for (int i = 0; i < HD; ++i) O[i] = 0.f;
            const int n0 = n;
            for (int t = sg.t0 + wg; t < sg.t1; t += 2, ++cnt) {
                const int nt = n0 + t - sg.t0;
                mbar_wait(&sh.sfull[wg], cnt & 1, a.err, ERR_WAIT_FULL, abort_flag);
                __syncwarp();
                tc_fence_after();
                const float f = KVT == KV_F16 ? qs : qs * pow2i(sh.ek[nt & 3]);
                const bool tail = (t + 1) * PT > s.n_ctx;
                // (the loops over 32-column chunks stay loops: unrolled, the code outgrows the
                // instruction cache and the one warp per scheduler waits for its fetches)
                float mx = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < PT / CH; ++c) {
                    uint32_t x[CH];
                    tmem_ld(ts + CH * c, x);
                    if (tail) {
                        const uint32_t vis = tree_window(a, s, sg.b, node, t * PT + CH * c - s.n_ctx);
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < CH; ++i) x[i] = (vis >> i) & 1 ? x[i] : 0xFF800000u;
                        tmem_st(ts + CH * c, x);  // masked scores are -infinity from here on
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
                for (int c = 0; c < PT / CH; ++c) {
                    uint32_t x[CH], y[CH];
                    tmem_ld(ts + CH * c, x);
#pragma unroll
                    for (int i = 0; i < CH; i += 2) {
                        const float p0 = exp2_fast(fmaf(__uint_as_float(x[i]), f, shift));
                        const float p1 = exp2_fast(fmaf(__uint_as_float(x[i + 1]), f, shift));
                        sum0 += p0;
                        sum1 += p1;
                        // high halves by truncation (exact in f16 down to 2^-14), low halves what is left
                        const float h0 = __uint_as_float(__float_as_uint(p0) & 0xFFFFE000u);
                        const float h1 = __uint_as_float(__float_as_uint(p1) & 0xFFFFE000u);
                        y[i / 2] = pack_half2(h0, h1);
                        y[CH / 2 + i / 2] = pack_half2(p0 - h0, p1 - h1);
                    }
                    tmem_st(ts + CH * c, y);
                }
                l = fmaf(l, alpha, sum0 + sum1);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&sh.pfull[wg]);
                mbar_wait(&sh.dfull[wg], cnt & 1, a.err, ERR_WAIT_FULL, abort_flag);
                __syncwarp();
                tc_fence_after();
                const float fv = KVT == KV_F16 ? 1.f : pow2i(sh.ev[nt & 3]);
#pragma unroll
                for (int c = 0; c < HD / CH; ++c) {
                    uint32_t x[CH];
                    tmem_ld(td + CH * c, x);
#pragma unroll
                    for (int i = 0; i < CH; ++i) O[CH * c + i] = fmaf(__uint_as_float(x[i]), fv, O[CH * c + i] * alpha);
                }
                tc_fence_before();
            }
            n += sg.t1 - sg.t0;
            // The streams meet in Q's shared memory (every QK of the segment is done): maxima and
            // sums first, then stream 1's weighted output, stream 0 adds its own, and the rows
            // leave coalesced.  fp32 rows of HD, 16-byte chunk c of row r at c ^ (r & 7).
            sh.ml[wg][row] = make_float2(m, l);
            named_bar<1, 256>();
            const float2 other = sh.ml[wg ^ 1][row];
            const float M = fmaxf(m, other.x), mref = M == -INFINITY ? 0.f : M, wgt = exp2_fast(m - mref);
            const float L = fmaf(l, wgt, other.y * exp2_fast(other.x - mref));
            const uint32_t srow = sb + F::Q_OFF + (uint32_t)row * (HD * 4);
            if (wg == 1) {
#pragma unroll
                for (int c = 0; c < HD / 4; ++c)
                    st_shared16(srow + ((uint32_t)(c ^ (row & 7)) << 4),
                                {__float_as_uint(O[4 * c] * wgt), __float_as_uint(O[4 * c + 1] * wgt),
                                 __float_as_uint(O[4 * c + 2] * wgt), __float_as_uint(O[4 * c + 3] * wgt)});
            }
            named_bar<1, 256>();
            const bool whole = sg.t0 == 0 && sg.t1 == sg.tiles;
            float* part = parts + ((size_t)blockIdx.x * 2 + (sg.t0 == 0 ? 1 : 0)) * tree_part_floats(TW_RT, hd);
            if (wg == 0) {
                const float inv = !whole ? 1.f : (L == 0.f ? 0.f : 1.f / L);
                const bool none = whole && L == 0.f;
#pragma unroll
                for (int c = 0; c < HD / 4; ++c) {
                    const uint32_t at = srow + ((uint32_t)(c ^ (row & 7)) << 4);
                    const uint4 x = ld_shared16(at);
                    const float y[4] = {fmaf(O[4 * c], wgt, __uint_as_float(x.x)), fmaf(O[4 * c + 1], wgt, __uint_as_float(x.y)),
                                        fmaf(O[4 * c + 2], wgt, __uint_as_float(x.z)), fmaf(O[4 * c + 3], wgt, __uint_as_float(x.w))};
                    uint32_t z[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) z[j] = none ? 0u : __float_as_uint(y[j] * inv);
                    st_shared16(at, z);
                }
                if (rr < rows) {
                    const size_t off = (size_t)s.slot * a.slot_stride + ((size_t)sg.kvh * a.cap + s.n_ctx) * hd;
#pragma unroll 1
                    for (int w = 0; w < TREE_MAX_NODES / 32; ++w)  // non-finite drafted values that the row sees
#pragma unroll 1
                        for (unsigned bits = sh.badrow[seg & 7][w] & tree_window(a, s, sg.b, node, 32 * w); bits; bits &= bits - 1) {
                            const size_t at = off + (size_t)(w * 32 + __ffs(bits) - 1) * hd;
#pragma unroll 1
                            for (int i = 0; i < hd; ++i) {
                                const float v = kv_load(a.vc, (long long)(at + i), KVT);
                                float* o = reinterpret_cast<float*>(smem + F::Q_OFF + (size_t)row * (HD * 4) + (((i >> 2) ^ (row & 7)) << 4)) + (i & 3);
                                if (!(fabsf(v) < INFINITY)) *o += v;
                            }
                        }
                    if (!whole && !*abort_flag) {
                        part[(size_t)TW_RT * hd + row] = M;
                        part[(size_t)TW_RT * hd + TW_RT + row] = L;
                    }
                }
                if (!whole && sg.t0 == 0 && row == 0) desc[blockIdx.x] = TreeDesc{sg.b, sg.kvh, sg.rtile, sg.last_cta};
            }
            named_bar<1, 256>();
            {
                constexpr int LPR = HD / 4, RPW = 32 / LPR;  // lanes per row, rows per warp and step
                const int c = lane % LPR;
#pragma unroll 4
                for (int i = warp; i < TW_RT / RPW; i += 8) {
                    const int r = i * RPW + lane / LPR, q = sg.rtile * TW_RT + r, nd = (q * rep_inv) >> 16;
                    if (q >= rows || c * 4 >= hd || *abort_flag) continue;
                    const uint4 x = ld_shared16(sb + F::Q_OFF + (uint32_t)r * (HD * 4) + ((uint32_t)(c ^ (r & 7)) << 4));
                    float* dst = whole ? a.out + ((size_t)sg.b * a.T + nd) * a.ld_out + (size_t)(sg.kvh * rep + q - nd * rep) * hd
                                       : part + (size_t)r * hd;
                    *reinterpret_cast<uint4*>(dst + c * 4) = x;
                }
            }
            named_bar<1, 256>();  // Q's shared memory takes the next segment's queries
            __syncwarp();
            ++seg;
        }
    }
    // TMEM stays allocated until every issued MMA has completed
    __syncwarp();
    if (warp == 0) mbar_wait(&sh.done, 0, a.err, ERR_WAIT_FULL, nullptr);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    tree_zero_rows<TW_THREADS>(a);
}

// ---- joins the partial results of units that were split over CTAs ------------------------------------
// Block (c, y): the unit that starts in CTA c's range and ends in a later one; a warp per row.
constexpr int TC_THREADS = 256;
__global__ void __launch_bounds__(TC_THREADS) tf_tree_combine_kernel(const TreeAttnArgs a, const TreePlan pl) {
    pdl_trigger();
    pdl_wait();
    const int c0 = blockIdx.x, lane = threadIdx.x & 31;
    const TreeDesc de = static_cast<const TreeDesc*>(a.ws)[c0];
    if (de.b < 0) return;
    const float* parts = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.ws) + 65536);
    const int rep = a.n_head / a.n_kv, hd = a.hd, rt = pl.rt, n = de.c1 - c0 + 1;
    const size_t pf = tree_part_floats(rt, hd);
    const int n_node = tree_seq(a, de.b).n_node;
    const int r = blockIdx.y * (TC_THREADS / 32) + (threadIdx.x >> 5), rr = de.rtile * rt + r;
    if (r >= rt || rr >= n_node * rep) return;
    auto part = [&](int i) { return parts + ((size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * pf; };
    float M = -INFINITY;
    for (int i = lane; i < n; i += 32) M = fmaxf(M, part(i)[(size_t)rt * hd + r]);
    M = warp_max(M);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const int d = lane * 4;
    for (int i0 = 0; i0 < n; i0 += 32) {
        float w = 0.f, lw = 0.f;
        if (i0 + lane < n) {
            const float* p = part(i0 + lane);
            w = exp2_fast(p[(size_t)rt * hd + r] - ref);
            lw = p[(size_t)rt * hd + rt + r] * w;
        }
        L += warp_sum(lw);
        const int k = min(32, n - i0);
#pragma unroll 4
        for (int i = 0; i < k; ++i) {
            const float wi = __shfl_sync(0xFFFFFFFFu, w, i);
            if (d < hd) {
                const float4 x = *reinterpret_cast<const float4*>(part(i0 + i) + (size_t)r * hd + d);
                o.x = fmaf(x.x, wi, o.x);
                o.y = fmaf(x.y, wi, o.y);
                o.z = fmaf(x.z, wi, o.z);
                o.w = fmaf(x.w, wi, o.w);
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

size_t tree_attn_ws_bytes(int B, int T, int n_head, int n_kv, int hd) {
    (void)B;
    const int rows = T * (n_head / n_kv), rt = rows <= 16 ? 16 : (rows <= 32 ? 32 : 64);
    return 65536 + (size_t)2 * tree_sms() * 2 * tree_part_floats(rt, hd) * sizeof(float);  // wide: half the CTAs, twice the rows
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
    pl.grid = 2 * tree_sms();
    pl.rt = F::RT;
    pl.pt = F::PT;
    pl.maps = 0;
    pl.min_tiles = 2;
    TreeAttnArgs aa = a;
    void* args[] = {&aa, &pl};
    cudaError_t e = tree_launch(fn, dim3(pl.grid), TN_THREADS, F::SMEM, args, st, pdl);
    if (e != cudaSuccess) return e;
    return tree_launch((const void*)tf_tree_combine_kernel, dim3(pl.grid, F::RT / (TC_THREADS / 32)), TC_THREADS, 0, args, st, true);
}

// The f16 cache as a 2-D tensor map: rows of hd halves, boxes of `pt` rows x 64 halves with the
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
    pl.grid = tree_sms();
    pl.rt = TW_RT;
    pl.pt = F::PT;
    pl.min_tiles = 2;
    alignas(64) CUtensorMap maps[2];
    memset(maps, 0, sizeof(maps));
    pl.maps = KVT == KV_F16 && a.hd == HD && tree_map(&maps[0], a, a.kc, F::PT) && tree_map(&maps[1], a, a.vc, F::PT);
    TreeAttnArgs aa = a;
    void* args[] = {&aa, &pl, &maps[0], &maps[1]};
    cudaError_t e = tree_launch(fn, dim3(pl.grid), TW_THREADS, F::SMEM, args, st, pdl);
    if (e != cudaSuccess) return e;
    return tree_launch((const void*)tf_tree_combine_kernel, dim3(pl.grid, TW_RT / (TC_THREADS / 32)), TC_THREADS, 0, args, st, true);
}

template <int HD, int KVT>
static cudaError_t narrow_rows(const TreeAttnArgs& a, cudaStream_t st, bool pdl) {
    const int rows = a.T * (a.n_head / a.n_kv);
    if (rows <= 16) return narrow_launch<HD, 1, KVT>(a, st, pdl);
    if (rows <= 32) return narrow_launch<HD, 2, KVT>(a, st, pdl);
    if (rows > 64) return wide_launch<HD, KVT>(a, st, pdl);
    return narrow_launch<HD, 4, KVT>(a, st, pdl);
}
template <int HD>
static cudaError_t narrow_type(const TreeAttnArgs& a, cudaStream_t st, bool pdl) {
    if (a.kv_type == KV_F32) return narrow_rows<HD, KV_F32>(a, st, pdl);
    if (a.kv_type == KV_F16) return narrow_rows<HD, KV_F16>(a, st, pdl);
    return narrow_rows<HD, KV_BF16>(a, st, pdl);
}

cudaError_t tree_attn_launch(const TreeAttnArgs& a, cudaStream_t st, bool pdl) {
    return a.hd <= 64 ? narrow_type<64>(a, st, pdl) : narrow_type<128>(a, st, pdl);
}

}  // namespace tfb
