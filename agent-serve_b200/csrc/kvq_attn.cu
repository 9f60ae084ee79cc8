// Attention over a quantised KV cache (Q4_0 / Q8_0, layout in kvq.cuh): T new rows per sequence, row t of
// sequence b seeing cache rows 0 .. n_ctx[b] + t; T = 1 is decode.
//
// Row (b, t, h): s_j = q . k_j / sqrt(hd), p_j = exp(s_j - max s), out = sum p_j v_j / sum p_j.
//
// Bound by the cache's bytes: a position of one kv head is 2 hd codes (144 bytes with its scales for 128 dims in
// 4 bits), so every warp instruction per position counts: at 6.5 TB/s an SM has 6.2 cycles for those 144 bytes,
// 25 issue slots.  Hence mma.sync m16n8k16 with the positions as M (K, then V transposed, is the A operand; a
// decode step has too few rows to fill M) and the rows as N, codes stored in the order of its fragments:
// a 32-bit word of eight codes is a shift, four LOP3 and four HADD2 away from four A registers, and no
// shared-memory pass or transpose is needed.  tcgen05 would want the codes unpacked through shared memory and 64 rows
// or more.
//
// Arithmetic (fp32-equivalent).  Codes less their zero are exact in f16: (code | 0x6400) is 1024 + code, and
// the high nibble in place 1024 + 16 code; the 16 is taken out of q (K) or of the output row (V).  q is split
// into two f16 halves after a power-of-two scale of its row (22 bits or more).  A group's products are summed from
// zero and enter the score by an fp32 fma with the group's scale.  V's scales multiply p (they differ by group of
// dims, so p is split once for each group): p = 2^(x - m + k), two f16 halves of p scale.  m is the row's
// running maximum, up to 2^8 behind; k comes from the largest V scale that the row has seen, so that p scale
// stays below 2^15 and its low half keeps 2^-24 / 2^7 of the largest; it is a row's own, since a row's bits must
// not hang on what only another row sees.
//
// Work is cut into units (sequence, kv head, row tile) and each unit into blocks of 16 positions; the
// blocks of all units, in order, are dealt out to the CTAs in equal contiguous ranges (lengths are read on the
// device), a CTA's warps take a range's blocks in turn, each with its own ring of cp.async copies (no barrier
// in the loop), and join at the range's end.  A unit that a range cuts leaves partial results for
// tf_kvq_combine_kernel, in a fixed order: results repeat bit for bit.
#include <atomic>

#include "kvq.cuh"

namespace tfb {

constexpr int KA_THREADS = 256;
constexpr int KA_WARPS = KA_THREADS / 32;
constexpr int KA_UNIT_COST = 8;    // blocks that a unit's start and end take the time of
constexpr int KA_SLACK = 8;        // binary orders that a running maximum may lag behind
constexpr int KA_MAX_GRID = 1024;  // descriptors of 16 bytes in the workspace's first 16 KB
constexpr size_t KA_DESC_BYTES = 16384;

struct KvqPlan {
    int grid;
    int rt;        // rows per row tile
    int rep;       // query heads per kv head
};
struct KvqDesc {   // a unit split over CTAs c0 .. c1, found at slot c0
    int b, kvh, tile, c1;  // b < 0: none; tile: row tile, and its rows in the high half
};

__host__ __device__ inline size_t kvq_part_floats(int rt, int hd) { return (size_t)rt * (hd + 2); }

// 0: up to 4 rows (both halves of q and p side by side in the 8 columns), 1: up to 8, 2: up to 16
__host__ __device__ constexpr int kvq_rt(int mode) { return mode == 0 ? 4 : mode == 1 ? 8 : 16; }

template <int BITS, int HD, int MODE>
struct KvqCfg {
    static constexpr int RT = kvq_rt(MODE);
    static constexpr int CTAS = MODE == 2 ? 1 : 2;                 // per SM
    static constexpr int BLOCK = kvq_block_bytes(BITS, HD);
    static constexpr int STAGE = 2 * BLOCK;                        // K and V of 16 positions
    static constexpr int SLOT = RT * HD * 4;                       // a warp's output rows
    static constexpr int STAT = KA_WARPS * RT * 8;
    static constexpr int ROOM = (CTAS == 2 ? 112 : 224) * 1024 - KA_WARPS * SLOT - STAT;
    static constexpr int FIT = ROOM / (KA_WARPS * STAGE);
    static constexpr int ST = FIT > 8 ? 8 : FIT;                   // stages of a warp's ring
    static constexpr int SMEM = KA_WARPS * (ST * STAGE + SLOT) + STAT;
    static_assert(ST >= 2, "two stages at least");
};

__device__ __forceinline__ float ka_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ka_mma(float (&c)[4], const uint32_t (&a)[4], const uint32_t b0, const uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t ka_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t ka_pack(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
__device__ __forceinline__ float2 ka_unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
// (1024 + u) in both halves -> u - z
template <int Z>
__device__ __forceinline__ uint32_t ka_centre(uint32_t x) {
    const __half2 y = __hadd2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(-1024.0f - Z));
    return *reinterpret_cast<const uint32_t*>(&y);
}
// the eight codes of a Q4_0 word, pairs 16 bits apart: codes 0 and 4, 1 and 5 (times 16), 2 and 6, 3 and 7 (times 16)
__device__ __forceinline__ void ka_nibbles(uint32_t w, uint32_t (&f)[4]) {
    const uint32_t v = w >> 8;
    f[0] = ka_centre<8>((w & 0x000F000Fu) | 0x64006400u);
    f[1] = ka_centre<128>((w & 0x00F000F0u) | 0x64006400u);
    f[2] = ka_centre<8>((v & 0x000F000Fu) | 0x64006400u);
    f[3] = ka_centre<128>((v & 0x00F000F0u) | 0x64006400u);
}
// the four codes of a Q8_0 word: codes 0 and 2, 1 and 3
__device__ __forceinline__ void ka_bytes(uint32_t w, uint32_t& f0, uint32_t& f1) {
    f0 = ka_centre<128>((w & 0x00FF00FFu) | 0x64006400u);
    f1 = ka_centre<128>((w >> 8 & 0x00FF00FFu) | 0x64006400u);
}
__device__ __forceinline__ void ka_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint32_t ka_lds(uint32_t at) {
    uint32_t x;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
    return x;
}
// N words that lie as kvq_word() places them for this lane
template <int N>
__device__ __forceinline__ void ka_words(uint32_t at, int lane, uint32_t (&w)[N]) {
#pragma unroll
    for (int c = 0; c < N / 4; ++c)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[4 * c]), "=r"(w[4 * c + 1]), "=r"(w[4 * c + 2]), "=r"(w[4 * c + 3])
                     : "r"(at + c * 512 + lane * 16)
                     : "memory");
    if (N % 4)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                     : "=r"(w[N - 2]), "=r"(w[N - 1])
                     : "r"(at + N / 4 * 512 + lane * 8)
                     : "memory");
}
// the scales of positions g and g + 8, HD / 32 groups each
template <int HD>
__device__ __forceinline__ void ka_scales(uint32_t at, int g, uint32_t (&s)[HD / 32]) {
    if (HD == 128)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(s[0]), "=r"(s[HD / 32 > 1 ? 1 : 0]), "=r"(s[HD / 32 > 2 ? 2 : 0]), "=r"(s[HD / 32 > 3 ? 3 : 0])
                     : "r"(at + g * 16)
                     : "memory");
    else
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) s[i] = ka_lds(at + g * (HD / 8) + 4 * i);
}
// scale of group k of position g (half 0) or g + 8 (half 1)
template <int N>
__device__ __forceinline__ float ka_scale(const uint32_t (&s)[N], int half, int k) {
    const int i = half * N + k;
    return h2f(i & 1 ? s[i >> 1] >> 16 : s[i >> 1]);
}

// ---- the split of the blocks over the CTAs ------------------------------------------------------------
struct KvqSeq {
    int slot, n_ctx, n_new, blocks, units;
    bool bad;
};
__device__ __forceinline__ KvqSeq kvq_seq(const KvqAttnArgs& a, const KvqPlan& pl, int b) {
    KvqSeq s;
    s.slot = a.slots ? a.slots[b] : b;
    s.n_ctx = a.n_ctx[b];
    s.n_new = a.n_new ? min(a.n_new[b], a.T) : a.T;
    s.bad = s.slot < 0 || s.slot >= a.n_slots || s.n_ctx < 0 || s.n_new < 0 || s.n_ctx > a.cap - s.n_new;
    if (s.bad) s.n_new = 0;
    s.blocks = s.n_new ? (s.n_ctx + s.n_new + 15) >> 4 : 0;
    s.units = a.n_kv * ((s.n_new * pl.rep + pl.rt - 1) / pl.rt);
    return s;
}
__device__ __forceinline__ int kvq_len(const KvqSeq& s) { return s.n_new ? s.units * (s.blocks + KA_UNIT_COST) : 0; }

// A CTA's range [g0, g1) of the flattened blocks: `b` is the sequence it begins in, `base` that one's start.
struct KvqRange {
    int g0, g1, per, b, base;
};
__device__ __forceinline__ KvqRange kvq_range(const KvqAttnArgs& a, const KvqPlan& pl) {
    const int lane = threadIdx.x & 31;
    const int chunk = (a.B + 31) >> 5, lo = min(a.B, lane * chunk), hi = min(a.B, lo + chunk);
    int mine = 0;
#pragma unroll 1
    for (int b = lo; b < hi; ++b) {
        const KvqSeq s = kvq_seq(a, pl, b);
        mine += kvq_len(s);
        if (s.bad && blockIdx.x == 0 && threadIdx.x < 32) atomicCAS(a.err, 0, ERR_POS);
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
    }
    const int total = __shfl_sync(0xFFFFFFFFu, inc, 31);
    KvqRange r;
    r.per = max(1, (int)(((unsigned)total + pl.grid - 1) / pl.grid));
    r.g0 = (int)min((long long)total, (long long)blockIdx.x * r.per);
    r.g1 = min(total, r.g0 + min(r.per, total - r.g0));
    const unsigned at = __ballot_sync(0xFFFFFFFFu, r.g0 >= inc - mine && r.g0 < inc);
    const int own = at ? __ffs(at) - 1 : 31;
    r.base = __shfl_sync(0xFFFFFFFFu, inc - mine, own);
    r.b = min(a.B, own * chunk);
    return r;
}

template <int BITS, int HD, int MODE>
__global__ void __launch_bounds__(KA_THREADS, KvqCfg<BITS, HD, MODE>::CTAS)
tf_kvq_attn_kernel(const KvqAttnArgs a, const KvqPlan pl) {
    using F = KvqCfg<BITS, HD, MODE>;
    constexpr int RT = F::RT, NT = MODE == 2 ? 2 : 1, NG = HD / 32, W = HD * BITS / 64, CODES = kvq_code_bytes(BITS, HD);
    constexpr int QP = MODE == 0 ? 1 : 2;  // parts of q and p that are products of their own
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    uint8_t* ring_p = smem + warp * (F::ST * F::STAGE);
    const uint32_t ring = smem_u32(ring_p);
    float* slot_all = reinterpret_cast<float*>(smem + KA_WARPS * F::ST * F::STAGE);
    float* stat = slot_all + KA_WARPS * RT * HD;  // [warp][RT] exponents, then sums
    KvqDesc* desc = static_cast<KvqDesc*>(a.ws);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + KA_DESC_BYTES);

    const KvqRange range = kvq_range(a, pl);
    KvqDesc open = {-1, 0, 0, 0};  // the unit that begins here and ends in a later CTA
    int b = range.b, base = range.base;
    const float log2e_d = 1.4426950408889634f * rsqrtf((float)HD);

#pragma unroll 1
    for (int gpos = range.g0; gpos < range.g1;) {
        KvqSeq sq = kvq_seq(a, pl, b);
        int len = kvq_len(sq);
        while (gpos >= base + len && b + 1 < a.B) {  // gpos is below the total: a sequence with work follows
            base += len;
            sq = kvq_seq(a, pl, ++b);
            len = kvq_len(sq);
        }
        if (gpos >= base + len) break;
        const int per_unit = sq.blocks + KA_UNIT_COST, unit = (gpos - base) / per_unit, ub = base + unit * per_unit;
        const int blk0 = gpos - ub, blk1 = min(sq.blocks, range.g1 - ub);
        gpos = min(range.g1, ub + per_unit);
        if (blk0 >= blk1) continue;
        const int tiles = sq.units / a.n_kv, kvh = unit / tiles, tile = unit - kvh * tiles;
        const int r0 = tile * RT, rows = min(RT, sq.n_new * pl.rep - r0);

        const long long where = sq.slot * a.slot_bytes + kvh * a.head_bytes;
        const uint8_t *kc = a.kc + where, *vc = a.vc + where;
        const int n_mine = blk1 - blk0 > warp ? (blk1 - blk0 - warp + KA_WARPS - 1) / KA_WARPS : 0;
        auto fetch = [&](int i) {  // block i of this warp's, in stage i % ST
            if (i < n_mine) {
                const long long off = (long long)(blk0 + warp + i * KA_WARPS) * F::BLOCK;
                const uint32_t dst = ring + i % F::ST * F::STAGE;
#pragma unroll
                for (int c = 0; c < (2 * F::BLOCK / 16 + 31) / 32; ++c) {
                    const int e = (c * 32 + lane) * 16;
                    if (e < F::BLOCK) ka_copy16(dst + e, kc + off + e);
                    else if (e < 2 * F::BLOCK) ka_copy16(dst + e, vc + off + (e - F::BLOCK));
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < F::ST - 1; ++i) fetch(i);

        // q as B fragments: column g is row g of the tile (packed: rows 0 .. 3 high, then rows 0 .. 3 low)
        uint32_t qf[NT][QP][NG][4];
        float fr[NT][2];  // of columns 2 tq and 2 tq + 1: out of q's scale, to powers of two
        int lim[NT][2];   // last position that they see
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = MODE == 0 ? g & 3 : nt * 8 + g, rr = r0 + row;
            const bool valid = row < rows;
            const int t = valid ? rr / pl.rep : 0, h = valid ? kvh * pl.rep + rr - t * pl.rep : 0;
            const float* qp = a.q + ((long long)b * a.T + t) * a.ld_q + h * HD + tq * 8;
            float x[NG][8], mx = 0.f;
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                const float4 u = valid ? *reinterpret_cast<const float4*>(qp + k * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float4 v = valid ? *reinterpret_cast<const float4*>(qp + k * 32 + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[k][0] = u.x; x[k][1] = u.y; x[k][2] = u.z; x[k][3] = u.w;
                x[k][4] = v.x; x[k][5] = v.y; x[k][6] = v.z; x[k][7] = v.w;
#pragma unroll
                for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[k][i]));
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
            // the row's largest value goes to [2^13, 2^14); rows of zeros, subnormals and infinities as they are
            const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
            const int sh = ex <= -127 || ex == 128 ? 0 : max(-120, min(120, 13 - ex));
            const float sc = __int_as_float((sh + 127) << 23);
            const float back = __int_as_float((127 - sh) << 23) * log2e_d;
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // codes 4 apart share a register in 4 bits (odd ones times 16), codes 2 apart in 8
                    const int e0 = BITS == 4 ? i : (i >> 1) * 4 + (i & 1), e1 = BITS == 4 ? i + 4 : e0 + 2;
                    const float down = BITS == 4 && (i & 1) ? sc * 0.0625f : sc;
                    const float u = x[k][e0] * down, v = x[k][e1] * down;
                    hi[i] = ka_pack(u, v);
                    const float2 f = ka_unpack(hi[i]);
                    lo[i] = ka_pack(u - f.x, v - f.y);
                    if (MODE == 0) qf[nt][0][k][i] = g < 4 ? hi[i] : lo[i];
                    else { qf[nt][0][k][i] = hi[i]; qf[nt][QP - 1][k][i] = lo[i]; }
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                fr[nt][j] = __shfl_sync(0xFFFFFFFFu, back, (2 * tq + j) * 4);
                const int c = MODE == 0 ? (2 * tq + j) & 3 : nt * 8 + 2 * tq + j;
                lim[nt][j] = sq.n_ctx + (r0 + c) / pl.rep;
            }
        }
        const int open_to = sq.n_ctx + r0 / pl.rep;  // every row sees the positions up to here

        float o[NT][HD / 16][4];
        float m[NT][2], ref[NT][2], l[NT][2];
        uint32_t top[NT][2];  // largest V scale that the column saw, rounded up within its binary order
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                m[nt][j] = -INFINITY;
                ref[nt][j] = 0.f;
                l[nt][j] = 0.f;
                top[nt][j] = 0;
            }
        }

#pragma unroll 1
        for (int i = 0; i < n_mine; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(F::ST - 2) : "memory");
            __syncwarp();  // everyone's copies of this stage are visible, and the stage before is read
            fetch(i + F::ST - 1);
            const uint32_t at = ring + i % F::ST * F::STAGE;
            const int p0 = (blk0 + warp + i * KA_WARPS) * 16;
            const bool masked = p0 + 15 > open_to;

            // scores: positions g and g + 8 (rows of C), columns 2 tq and 2 tq + 1
            float x[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
            {
                uint32_t w[W], s[NG];
                ka_words<W>(at, lane, w);
                ka_scales<HD>(at + CODES, g, s);
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    uint32_t a0[4], a1[4];
                    if (BITS == 4) {
                        uint32_t u[4], v[4];
                        ka_nibbles(w[k], u);
                        ka_nibbles(w[W / 2 + k], v);
                        a0[0] = u[0]; a0[1] = v[0]; a0[2] = u[1]; a0[3] = v[1];
                        a1[0] = u[2]; a1[1] = v[2]; a1[2] = u[3]; a1[3] = v[3];
                    } else {
                        ka_bytes(w[2 * k], a0[0], a0[2]);
                        ka_bytes(w[W / 2 + 2 * k], a0[1], a0[3]);
                        ka_bytes(w[2 * k + 1], a1[0], a1[2]);
                        ka_bytes(w[W / 2 + 2 * k + 1], a1[1], a1[3]);
                    }
                    const float s0 = ka_scale(s, 0, k), s1 = ka_scale(s, 1, k);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int part = QP - 1; part >= 0; --part) {  // the low halves first
                            ka_mma(c, a0, qf[nt][part][k][0], qf[nt][part][k][1]);
                            ka_mma(c, a1, qf[nt][part][k][2], qf[nt][part][k][3]);
                        }
                        x[nt][0] = fmaf(c[0], s0, x[nt][0]);
                        x[nt][1] = fmaf(c[1], s0, x[nt][1]);
                        x[nt][2] = fmaf(c[2], s1, x[nt][2]);
                        x[nt][3] = fmaf(c[3], s1, x[nt][3]);
                    }
                }
            }
            if (MODE == 0) {  // column c holds the high half's part of row c, column c + 4 the low half's
#pragma unroll
                for (int e = 0; e < 4; ++e) x[0][e] += __shfl_xor_sync(0xFFFFFFFFu, x[0][e], 2);
            }
            uint32_t vs[NG];
            ka_scales<HD>(at + F::BLOCK + CODES, g, vs);
            // largest |scale| of V at positions g and g + 8; NaN and infinity have no say
            uint32_t big0 = 0, big1 = 0;
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                const int i0 = k, i1 = NG + k;
                const uint32_t e0 = (i0 & 1 ? vs[i0 >> 1] >> 16 : vs[i0 >> 1]) & 0x7FFFu;
                const uint32_t e1 = (i1 & 1 ? vs[i1 >> 1] >> 16 : vs[i1 >> 1]) & 0x7FFFu;
                if (e0 < 0x7C00u) big0 = max(big0, e0);
                if (e1 < 0x7C00u) big1 = max(big1, e1);
            }
            bool raise = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = e & 1;
                    const bool seen = !masked || p0 + g + (e >> 1) * 8 <= lim[nt][j];
                    x[nt][e] = seen ? x[nt][e] * fr[nt][j] : -INFINITY;
                    raise |= x[nt][e] > m[nt][j] + (float)KA_SLACK || (seen && (e >> 1 ? big1 : big0) > top[nt][j]);
                }
            if (__any_sync(0xFFFFFFFFu, raise)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float mx = fmaxf(m[nt][j], fmaxf(x[nt][j], x[nt][2 + j]));
                        uint32_t tp = top[nt][j];
                        if (!masked || p0 + g <= lim[nt][j]) tp = max(tp, big0);
                        if (!masked || p0 + g + 8 <= lim[nt][j]) tp = max(tp, big1);
#pragma unroll
                        for (int s = 4; s < 32; s <<= 1) {
                            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, s));
                            tp = max(tp, __shfl_xor_sync(0xFFFFFFFFu, tp, s));
                        }
                        // a column moves by what it sees alone, whichever column asked
                        const bool move = mx > m[nt][j] + (float)KA_SLACK || tp > top[nt][j];
                        if (!move) continue;
                        tp |= 0x3FFu;  // scales are below 2^(tp / 1024 - 14)
                        const float nref = mx == -INFINITY ? 0.f : mx - (float)(15 - KA_SLACK + 14 - (int)(tp >> 10));
                        const float f = m[nt][j] == -INFINITY ? 0.f : ka_exp2(ref[nt][j] - nref);
                        // (a row that saw nothing yet has sums of zero, or NaN, which stays)
                        m[nt][j] = mx;
                        ref[nt][j] = nref;
                        top[nt][j] = tp;
                        l[nt][j] *= f;
#pragma unroll
                        for (int d = 0; d < HD / 16; ++d) {
                            o[nt][d][j] *= f;
                            o[nt][d][2 + j] *= f;
                        }
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[nt][e] = ka_exp2(x[nt][e] - ref[nt][e & 1]);
                    l[nt][e & 1] += x[nt][e];
                }
            uint32_t w[W];
            ka_words<W>(at + F::BLOCK, lane, w);
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                const float s0 = ka_scale(vs, 0, k), s1 = ka_scale(vs, 1, k);
                uint32_t pf[NT][QP][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float y[4] = {x[nt][0] * s0, x[nt][1] * s0, x[nt][2] * s1, x[nt][3] * s1};
                    if (masked) {  // an unseen position's scale may be NaN
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (p0 + g + (e >> 1) * 8 > lim[nt][e & 1]) y[e] = 0.f;
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t hi = ka_pack(y[2 * e], y[2 * e + 1]);
                        const float2 f = ka_unpack(hi);
                        const uint32_t lo = ka_pack(y[2 * e] - f.x, y[2 * e + 1] - f.y);
                        if (MODE == 0) {
                            pf[nt][0][e] = ka_trans(tq < 2 ? hi : lo);
                        } else {
                            pf[nt][0][e] = ka_trans(hi);
                            pf[nt][QP - 1][e] = ka_trans(lo);
                        }
                    }
                }
#pragma unroll
                for (int d = 2 * k; d < 2 * k + 2; ++d) {
                    uint32_t v[4];
                    if (BITS == 4) {
                        ka_nibbles(w[d], v);
                    } else {
                        ka_bytes(w[2 * d], v[0], v[2]);
                        ka_bytes(w[2 * d + 1], v[1], v[3]);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int part = QP - 1; part >= 0; --part) ka_mma(o[nt][d], v, pf[nt][part][0], pf[nt][part][1]);
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // the warp's rows into its slot: dims 16 d + 2 g and one on, rows 2 tq and one on
        __syncthreads();  // the slots of the segment before are read
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int s = 4; s < 32; s <<= 1) l[nt][j] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][j], s);
                const int row = nt * 8 + 2 * tq + j;
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) {
                    float2 y = make_float2(o[nt][d][j], o[nt][d][2 + j] * (BITS == 4 ? 0.0625f : 1.0f));
                    if (MODE == 0) {
                        y.x += __shfl_xor_sync(0xFFFFFFFFu, y.x, 2);
                        y.y += __shfl_xor_sync(0xFFFFFFFFu, y.y, 2);
                    }
                    if (row < RT) *reinterpret_cast<float2*>(slot_all + (warp * RT + row) * HD + 16 * d + 2 * g) = y;
                }
                if (g == 0 && row < RT) {
                    // a warp without blocks, or whose rows saw nothing: its exponent says so
                    const bool none = n_mine == 0 || (m[nt][j] == -INFINITY && l[nt][j] == 0.f);
                    stat[warp * RT + row] = none ? -INFINITY : ref[nt][j];
                    stat[(KA_WARPS + warp) * RT + row] = l[nt][j];
                }
            }
        __syncthreads();
        const bool begins = blk0 == 0, ends = blk1 == sq.blocks;
        float* part = parts + (blockIdx.x * 2 + (begins ? 1 : 0)) * kvq_part_floats(RT, HD);
        for (int i = threadIdx.x; i < rows * (HD / 4); i += KA_THREADS) {
            const int row = i / (HD / 4), d = (i - row * (HD / 4)) * 4;
            float mx = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < KA_WARPS; ++w) mx = fmaxf(mx, stat[w * RT + row]);
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < KA_WARPS; ++w) {
                const float e = stat[w * RT + row];
                if (e == -INFINITY) continue;
                const float f = ka_exp2(e - mx);
                const float4 u = *reinterpret_cast<const float4*>(slot_all + (w * RT + row) * HD + d);
                L = fmaf(stat[(KA_WARPS + w) * RT + row], f, L);
                y.x = fmaf(u.x, f, y.x);
                y.y = fmaf(u.y, f, y.y);
                y.z = fmaf(u.z, f, y.z);
                y.w = fmaf(u.w, f, y.w);
            }
            if (begins && ends) {
                const int rr = r0 + row, t = rr / pl.rep, h = kvh * pl.rep + rr - t * pl.rep;
                const float inv = L == 0.f ? 0.f : 1.0f / L;
                *reinterpret_cast<float4*>(a.out + ((long long)b * a.T + t) * a.ld_out + h * HD + d) =
                    make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
            } else {
                *reinterpret_cast<float4*>(part + row * HD + d) = y;
                if (d == 0) {
                    part[RT * HD + row] = mx;
                    part[RT * HD + RT + row] = L;
                }
            }
        }
        if (begins && !ends) open = KvqDesc{b, kvh, tile | rows << 16, (ub + sq.blocks - 1) / range.per};
    }
    if (threadIdx.x == 0) desc[blockIdx.x] = open;

    // rows behind a sequence's new ones, and rows of a sequence that was refused, are zero
    for (int s = blockIdx.x; s < a.B; s += pl.grid) {
        const KvqSeq sq = kvq_seq(a, pl, s);
        const int n = a.n_head * HD / 4;
        for (int t = sq.n_new; t < a.T; ++t)
            for (int i = threadIdx.x; i < n; i += KA_THREADS)
                *reinterpret_cast<float4*>(a.out + ((long long)s * a.T + t) * a.ld_out + i * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
}

// ---- joins the partial results of units that were split over CTAs ------------------------------------
// Block (c, y): the unit that begins in CTA c's range and ends in a later one; a warp per row.
constexpr int KC_WARPS = 4;
__global__ void __launch_bounds__(KC_WARPS * 32) tf_kvq_combine_kernel(const KvqAttnArgs a, const KvqPlan pl) {
    pdl_wait();
    const int c0 = blockIdx.x, lane = threadIdx.x & 31, r = blockIdx.y * KC_WARPS + (threadIdx.x >> 5);
    const KvqDesc de = static_cast<const KvqDesc*>(a.ws)[c0];
    if (de.b < 0 || r >= de.tile >> 16) return;
    const float* parts = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.ws) + KA_DESC_BYTES);
    const int hd = a.hd, rt = pl.rt, n = de.c1 - c0 + 1, d = lane * 4;
    const size_t pf = kvq_part_floats(rt, hd);
    auto part = [&](int i) { return parts + ((size_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * pf; };
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 32) {  // 32 parts at a time, eight parts' rows in flight
        const int k = min(32, n - i0);
        float m = -INFINITY, l = 0.f;
        if (lane < k) {
            const float* p = part(i0 + lane) + (size_t)rt * hd + r;
            m = p[0];
            l = p[rt];
        }
        const float mx = fmaxf(M, warp_max(m)), at = mx == -INFINITY ? 0.f : mx;
        const float alpha = ka_exp2(M - at), w = m == -INFINITY ? 0.f : ka_exp2(m - at);
        M = mx;
        L = fmaf(L, alpha, warp_sum(m == -INFINITY ? 0.f : l * w));
        o = make_float4(o.x * alpha, o.y * alpha, o.z * alpha, o.w * alpha);
#pragma unroll 1
        for (int i = 0; i < k; i += 8) {
            float4 x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = i + j < k && d < hd ? *reinterpret_cast<const float4*>(part(i0 + i + j) + (size_t)r * hd + d)
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
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
    if (d >= hd) return;
    const int rep = pl.rep, rr = (de.tile & 0xFFFF) * rt + r, t = rr / rep, h = de.kvh * rep + rr - t * rep;
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    *reinterpret_cast<float4*>(a.out + ((long long)de.b * a.T + t) * a.ld_out + h * hd + d) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// ---- host ------------------------------------------------------------------------------------------
static int kvq_sms() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms < 1 ? 1 : (2 * sms > KA_MAX_GRID ? KA_MAX_GRID / 2 : sms);
}
static int kvq_mode(int rows) { return rows <= 4 ? 0 : rows <= 8 ? 1 : 2; }

size_t kvq_attn_ws_bytes(int T, int n_head, int n_kv, int hd) {
    const int mode = kvq_mode(T * (n_head / n_kv));
    return KA_DESC_BYTES + (size_t)kvq_sms() * (mode == 2 ? 1 : 2) * 2 * kvq_part_floats(kvq_rt(mode), hd) * sizeof(float);
}

// Units of 4 rows or more, blocks of 16 positions and a unit's cost.
bool kvq_attn_fits(int B, int T, int n_head, int n_kv, int cap) {
    const int rows = T * (n_head / n_kv), rt = kvq_rt(kvq_mode(rows));
    return (double)B * n_kv * ((rows + rt - 1) / rt) * ((double)cap / 16 + KA_UNIT_COST) < 2147483648.0;
}

static cudaError_t kvq_launch(const void* fn, dim3 grid, int threads, size_t smem, void** args, cudaStream_t st, bool pdl) {
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

template <int BITS, int HD, int MODE>
static cudaError_t mode_launch(const KvqAttnArgs& a, cudaStream_t st) {
    using F = KvqCfg<BITS, HD, MODE>;
    const void* fn = (const void*)tf_kvq_attn_kernel<BITS, HD, MODE>;
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
    KvqPlan pl;
    pl.grid = kvq_sms() * F::CTAS;
    pl.rt = F::RT;
    pl.rep = a.n_head / a.n_kv;
    KvqAttnArgs aa = a;
    void* args[] = {&aa, &pl};
    cudaError_t e = kvq_launch(fn, dim3(pl.grid), KA_THREADS, F::SMEM, args, st, false);
    if (e != cudaSuccess) return e;
    return kvq_launch((const void*)tf_kvq_combine_kernel, dim3(pl.grid, F::RT / KC_WARPS), KC_WARPS * 32, 0, args, st, true);
}
template <int BITS, int HD>
static cudaError_t hd_launch(const KvqAttnArgs& a, cudaStream_t st) {
    const int mode = kvq_mode(a.T * (a.n_head / a.n_kv));
    return mode == 0 ? mode_launch<BITS, HD, 0>(a, st) : mode == 1 ? mode_launch<BITS, HD, 1>(a, st) : mode_launch<BITS, HD, 2>(a, st);
}
template <int BITS>
static cudaError_t bits_launch(const KvqAttnArgs& a, cudaStream_t st) {
    if (a.hd == 32) return hd_launch<BITS, 32>(a, st);
    if (a.hd == 64) return hd_launch<BITS, 64>(a, st);
    if (a.hd == 96) return hd_launch<BITS, 96>(a, st);
    return a.hd == 128 ? hd_launch<BITS, 128>(a, st) : cudaErrorInvalidValue;
}

cudaError_t kvq_attn_launch(const KvqAttnArgs& a, cudaStream_t st) {
    if (!kvq_attn_fits(a.B, a.T, a.n_head, a.n_kv, a.cap)) return cudaErrorInvalidValue;
    return a.bits == 4 ? bits_launch<4>(a, st) : bits_launch<8>(a, st);
}

}  // namespace tfb
