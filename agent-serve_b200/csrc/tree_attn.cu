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
#include <atomic>

#include "tree.cuh"

namespace tfb {

constexpr int TN_THREADS = 256;
constexpr int TN_TILE_BYTES = 32768;  // K and V bytes of a tile in the cache's type: 32 registers per thread
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 15.f;       // p is held as 2^15 exp(s - max): its low half keeps 2^-24 / 2^15 of it

// ---- the split of the tiles over the CTAs ---------------------------------------------------------
struct TreePlan {
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

    while (g0 < g1) {
        TreeSeq s = tree_seq(a, b);
        int tiles = seq_tiles(s, PT), units = seq_units(a, s, RT);
        while (g0 >= base + (long long)tiles * units) {  // next sequence with work
            base += (long long)tiles * units;
            s = tree_seq(a, ++b);
            tiles = seq_tiles(s, PT);
            units = seq_units(a, s, RT);
        }
        const int unit = (int)((g0 - base) / tiles), nrt = units / a.n_kv;
        const int kvh = unit / nrt, rtile = unit % nrt;
        const long long u0 = base + (long long)unit * tiles;  // the unit's first tile
        const int t0 = (int)(g0 - u0), t1 = (int)(g1 - u0 < tiles ? g1 - u0 : tiles);
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
            constexpr int TPR = TN_THREADS / RT < HD / 8 ? TN_THREADS / RT : HD / 8, EPT = HD / TPR;
            const int r = tid / TPR, rr = rtile * RT + r, d0 = (tid % TPR) * EPT;
            if (r < RT) {
                float x[EPT];
                uint32_t mb = 0;
                const int node = div_rep(rr);
                const float* qp = a.q + ((size_t)b * a.T + node) * a.ld_q + (size_t)(kvh * rep + rr - node * rep) * hd;
#pragma unroll
                for (int i = 0; i < EPT; i += 4) {
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (rr < rows && d0 + i < hd) y = *reinterpret_cast<const float4*>(qp + d0 + i);
                    x[i] = y.x, x[i + 1] = y.y, x[i + 2] = y.z, x[i + 3] = y.w;
                }
#pragma unroll
                for (int i = 0; i < EPT; ++i) mb = max(mb, finite_abs_bits(x[i]));
#pragma unroll
                for (int o = 1; o < TPR; o <<= 1) mb = max(mb, __shfl_xor_sync(0xFFFFFFFFu, mb, o));
                const int e = half_exponent(mb);
                const float sc = pow2i(-e);
#pragma unroll
                for (int i = 0; i < EPT; i += 8) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) split2(x[i + 2 * j] * sc, x[i + 2 * j + 1] * sc, hi[j], lo[j]);
                    const uint32_t c = (uint32_t)(d0 + i) >> 3;
                    const uint32_t o = (uint32_t)r * (HD * 2) + ((c ^ (r & 7)) << 4);
                    st_shared16(qh + o, hi);
                    st_shared16(ql + o, lo);
                }
                if (d0 == 0) qscale[r] = pow2i(e) * (kLog2e / sqrtf((float)hd));
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
        const bool whole = t0 == 0 && t1 == tiles;
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
            desc[blockIdx.x] = TreeDesc{b, kvh, rtile, (int)((u0 + tiles - 1) / per)};
        g0 = u0 + t1;
        __syncthreads();
    }
    tree_zero_rows<TN_THREADS>(a);
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
    return 65536 + (size_t)2 * tree_sms() * 2 * tree_part_floats(rt, hd) * sizeof(float);
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
    pl.min_tiles = 2;
    TreeAttnArgs aa = a;
    void* args[] = {&aa, &pl};
    cudaError_t e = tree_launch(fn, dim3(pl.grid), TN_THREADS, F::SMEM, args, st, pdl);
    if (e != cudaSuccess) return e;
    return tree_launch((const void*)tf_tree_combine_kernel, dim3(pl.grid, F::RT / (TC_THREADS / 32)), TC_THREADS, 0, args, st, true);
}

template <int HD, int KVT>
static cudaError_t narrow_rows(const TreeAttnArgs& a, cudaStream_t st, bool pdl) {
    const int rows = a.T * (a.n_head / a.n_kv);
    if (rows <= 16) return narrow_launch<HD, 1, KVT>(a, st, pdl);
    if (rows <= 32) return narrow_launch<HD, 2, KVT>(a, st, pdl);
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
