// Attention over a quantised KV cache (Q4_0 / Q8_0, layout in kvq.cuh): T new rows per sequence, row t of
// sequence b seeing cache rows 0 .. n_ctx[b] + t; T = 1 is decode.
//
// Row (b, t, h): s_j = q . k_j / sqrt(hd), p_j = exp(s_j - max s), out = sum p_j v_j / sum p_j.
//
// Bound by the cache's bytes: a position of one kv head is 2 hd codes (144 bytes with its scales for 128 dims in
// 4 bits), so every warp instruction per position counts: at 6.5 TB/s an SM has 6.2 cycles for those 144 bytes,
// 25 issue slots.  Hence mma.sync m16n8k16 with the codes in the order of its fragments: a 32-bit word of eight
// codes is a shift, four LOP3 and four HADD2 away from four operand registers, and no shared-memory pass or
// transpose is needed.  Scores have the rows as M and the positions as N (K is the B operand), the second product
// the dims as M and the rows as N (V transposed is the A operand), so that the scores' registers are the
// probabilities' operand as they stand.  Up to 8 rows, the M of 16 holds q's high and low halves; up to 4, the N of 8
// holds p's.  tcgen05 would want the codes unpacked through shared memory and 64 rows or more.
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
#include <type_traits>

#include "kvq.cuh"

namespace tfb {

constexpr int KA_THREADS = 128;
constexpr int KA_WARPS = KA_THREADS / 32;
constexpr int KA_UNIT_COST = 8;    // blocks that a unit's start and end take the time of
constexpr int KA_MIN_RANGE = 16;   // blocks of a CTA's range at least
constexpr int KA_MAX_SPLIT = 8;    // CTAs of a cluster
constexpr int KA_SNAP = 6;         // a cut this near to a unit's first or last block moves there
constexpr int KA_SLACK = 8;        // binary orders that a running maximum may lag behind
constexpr int KA_MAX_GRID = 1024;  // descriptors of 32 bytes in the workspace's first 32 KB
constexpr size_t KA_DESC_BYTES = 32768;

struct KvqPlan {
    int grid;
    int rt;        // rows per row tile
    int rep;       // query heads per kv head
    int tiles;     // row tiles of T rows
    int split;     // CTAs of a unit, one cluster; 0: ranges of all units' blocks
    int by_unit;   // descriptors are found by unit (there are at most `grid`), else by the CTA that begins it
};
struct alignas(32) KvqDesc {  // a unit split over CTAs c0 .. c1
    int b, kvh, tile, rows, c0, c1;  // b < 0: no unit, or one that was not split
};

__host__ __device__ inline size_t kvq_part_floats(int rt, int hd) { return (size_t)rt * (hd + 2); }

// 0: up to 4 rows (both halves of q and p side by side in the 8 columns), 1: up to 8, 2: up to 16
__host__ __device__ constexpr int kvq_rt(int mode) { return mode == 0 ? 4 : mode == 1 ? 8 : 16; }

__host__ __device__ constexpr int kvq_ctas(int mode) { return mode == 2 ? 3 : 4; }  // 168 or 128 registers a thread

template <int BITS, int HD, int MODE>
struct KvqCfg {
    static constexpr int RT = kvq_rt(MODE);
    static constexpr int CTAS = kvq_ctas(MODE);                    // per SM
    static constexpr int BLOCK = kvq_block_bytes(BITS, HD);
    static constexpr int SLOT = RT * HD * 4;                       // a warp's output rows
    static constexpr int QF = (MODE == 2 ? 2 : 1) * HD / 32 * 1024;  // q's fragments
    static constexpr int STAT = KA_WARPS * RT * 12;
    static constexpr int ROOM = 227 * 1024 / CTAS - 1024 - STAT - QF;
    static constexpr int PB = HD < 128 && ROOM >= 8 * KA_WARPS * BLOCK ? 2 : 1;  // neighbouring blocks of a warp's turn: two where two stages fit
    static constexpr int STAGE = 2 * PB * BLOCK;                   // K, then V
    static constexpr int FIT = ROOM / (KA_WARPS * STAGE);
    static constexpr int ST = FIT > 8 ? 8 : FIT;                   // stages of a warp's ring
    static constexpr int RING = ST * STAGE > SLOT ? ST * STAGE : SLOT;  // output rows take the rings' place
    static constexpr int SMEM = KA_WARPS * RING + STAT + QF;
    static_assert(ST >= 2 && KA_WARPS * RING + STAT + QF <= 227 * 1024 / CTAS - 1024, "two stages at least");
};

__device__ __forceinline__ float ka_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ka_mma(float (&c)[4], const uint32_t (&a)[4], const uint32_t b0, const uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t ka_pack_rz(float lo, float hi) {  // towards zero
    uint32_t y;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
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
// (w & MASK) | magic in one instruction: of two constants one has to lie in a register, which the caller sees to
template <uint32_t MASK>
__device__ __forceinline__ uint32_t ka_field(uint32_t w, uint32_t magic) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(w), "n"(MASK), "r"(magic));
    return y;
}
// the eight codes of a Q4_0 word, pairs 16 bits apart: codes 0 and 4, 1 and 5 (times 16), 2 and 6, 3 and 7 (times 16)
__device__ __forceinline__ void ka_nibbles(uint32_t w, uint32_t magic, uint32_t (&f)[4]) {
    const uint32_t v = w >> 8;
    f[0] = ka_centre<8>(ka_field<0x000F000Fu>(w, magic));
    f[1] = ka_centre<128>(ka_field<0x00F000F0u>(w, magic));
    f[2] = ka_centre<8>(ka_field<0x000F000Fu>(v, magic));
    f[3] = ka_centre<128>(ka_field<0x00F000F0u>(v, magic));
}
// the four codes of a Q8_0 word: codes 0 and 2, 1 and 3
__device__ __forceinline__ void ka_bytes(uint32_t w, uint32_t magic, uint32_t& f0, uint32_t& f1) {
    f0 = ka_centre<128>(ka_field<0x00FF00FFu>(w, magic));
    f1 = ka_centre<128>(ka_field<0x00FF00FFu>(w >> 8, magic));
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 ka_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
        "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 ka_mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
        "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ void ka_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ka_lds4(const uint8_t* p, uint32_t* x) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    x[0] = v.x;
    x[1] = v.y;
    x[2] = v.z;
    x[3] = v.w;
}
__device__ __forceinline__ void ka_lds2(const uint8_t* p, uint32_t* x) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = v.x;
    x[1] = v.y;
}
// N words that lie as kvq_word() places them for this lane
template <int N>
__device__ __forceinline__ void ka_words(const uint8_t* p, int lane, uint32_t (&w)[N]) {
#pragma unroll
    for (int c = 0; c < N / 4; ++c) ka_lds4(p + c * 512 + lane * 16, &w[4 * c]);
    if (N % 4) ka_lds2(p + N / 4 * 512 + lane * 8, &w[N - 2]);
}
// the scales of positions 2 tq, 2 tq + 8, 2 tq + 1, 2 tq + 9: NG = HD / 32 groups each, two to a word
template <int NG>
__device__ __forceinline__ void ka_scales(const uint8_t* p, int tq, uint32_t (&s)[2 * NG]) {
#pragma unroll
    for (int i = 0; i < 2 * NG; i += NG % 2 ? 2 : 4) {
        if (NG % 2) ka_lds2(p + tq * (8 * NG) + 4 * i, &s[i]);
        else ka_lds4(p + tq * (8 * NG) + 4 * i, &s[i]);
    }
}
// Scale of group k of position 2 tq + e (e = 0, 1) or 2 tq + 8 + e - 2 (e = 2, 3).
template <int N>
__device__ __forceinline__ float ka_scale(const uint32_t (&s)[N], int e, int k) {
    const int i = ((e & 1) * 2 + (e >> 1)) * (N / 2) + k;
    const __half2 h = *reinterpret_cast<const __half2*>(&s[i >> 1]);
    return i & 1 ? __high2float(h) : __low2float(h);
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

// Where the cut at offset t of a unit of n blocks falls: near a unit's ends it would cost a partial result for
// next to nothing.
__device__ __forceinline__ int kvq_cut(int t, int n) { return t < KA_SNAP ? 0 : n - t < KA_SNAP ? max(t, n) : t; }

// A CTA's range [g0, g1) of the flattened blocks, before its ends are moved (kvq_cut): `b` is the sequence it
// begins in, `base` that one's start.
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
    r.per = max(KA_MIN_RANGE, (int)(((unsigned)total + pl.grid - 1) / pl.grid));
    r.g0 = (int)min((long long)total, (long long)blockIdx.x * r.per);
    r.g1 = min(total, r.g0 + min(r.per, total - r.g0));
    const unsigned at = __ballot_sync(0xFFFFFFFFu, r.g0 >= inc - mine && r.g0 < inc);
    const int own = at ? __ffs(at) - 1 : 31;
    r.base = __shfl_sync(0xFFFFFFFFu, inc - mine, own);
    r.b = min(a.B, own * chunk);
    return r;
}

// Every thread of the cluster arrives; shared memory written before is visible after.
__device__ __forceinline__ void ka_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t ka_remote(const void* p, int rank) {  // the same place in another CTA of the cluster
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float ka_remote1(const float* p, int rank) {
    float x;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(ka_remote(p, rank)) : "memory");
    return x;
}
__device__ __forceinline__ float4 ka_remote4(const float* p, int rank) {
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                 : "r"(ka_remote(p, rank))
                 : "memory");
    return x;
}

// CLUSTER: a cluster of pl.split CTAs per unit (all of them, from the sequences' T rows), which join over distributed
// shared memory; else ranges, and a second launch.
template <int BITS, int HD, int MODE, bool CLUSTER>
__global__ void __launch_bounds__(KA_THREADS, KvqCfg<BITS, HD, MODE>::CTAS)
tf_kvq_attn_kernel(const KvqAttnArgs a, const KvqPlan pl) {
    using F = KvqCfg<BITS, HD, MODE>;
    constexpr int RT = F::RT, NG = HD / 32, W = HD * BITS / 64, CODES = kvq_code_bytes(BITS, HD);
    constexpr int NR = MODE == 2 ? 2 : 1;  // rows of a thread: g, and g + 8
    constexpr int QP = MODE == 2 ? 2 : 1;  // products of q's halves: side by side in M, or one after the other
    constexpr int PP = MODE == 0 ? 1 : 2;  // products of p's halves: side by side in N, or one after the other
    extern __shared__ __align__(128) uint8_t smem[];
    if (!CLUSTER) pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    const uint32_t ring_at = warp * (F::ST * F::STAGE), ring = smem_u32(smem) + ring_at;
    uint8_t* qs = smem + KA_WARPS * F::RING;  // [QP][NG][2][lane] four registers
    const uint8_t* q_at = qs + lane * 16;
    float* slot_all = reinterpret_cast<float*>(smem);  // where the rings are, once a segment's blocks are done
    float* stat = reinterpret_cast<float*>(qs + F::QF);  // [warp][RT] exponents, then sums, then q's maxima
    float* q_max = stat + 2 * KA_WARPS * RT;
    KvqDesc* desc = static_cast<KvqDesc*>(a.ws);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + KA_DESC_BYTES);

    KvqRange range = {0, 1, 0, 0, 0};
    int b = 0, base = 0, rank = 0;
    if (CLUSTER) {
        rank = blockIdx.x % pl.split;
        b = blockIdx.x / (pl.split * pl.tiles * a.n_kv);
    } else {
        range = kvq_range(a, pl);
        b = range.b;
        base = range.base;
    }
    KvqDesc open = {-1, 0, 0, 0, 0, 0};  // the unit that begins here and ends in a later CTA
    const float log2e_d = 1.4426950408889634f * rsqrtf((float)HD);
    uint32_t magic;
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));

#pragma unroll 1
    for (int gpos = range.g0; gpos < range.g1;) {
        KvqSeq sq = kvq_seq(a, pl, b);
        int blk0, blk1, kvh, tile, rows, r0, ub = 0;
        if (CLUSTER) {
            gpos = range.g1;
            const int unit = blockIdx.x / pl.split - b * (pl.tiles * a.n_kv);
            kvh = unit / pl.tiles;
            tile = unit - kvh * pl.tiles;
            if (sq.bad && unit == 0 && rank == 0 && threadIdx.x == 0) atomicCAS(a.err, 0, ERR_POS);
            const int each = (sq.blocks + pl.split - 1) / pl.split;
            blk0 = min(rank * each, sq.blocks);
            blk1 = min(blk0 + each, sq.blocks);
            r0 = tile * RT;
            // the tile's rows behind the new ones are zero
            const int all = min(RT, a.T * pl.rep - r0), first = max(0, sq.n_new * pl.rep - r0);
            for (int i = first * (HD / 4) + rank * KA_THREADS + threadIdx.x; i < all * (HD / 4); i += pl.split * KA_THREADS) {
                const int row = i / (HD / 4), rr = r0 + row, t = rr / pl.rep, h = kvh * pl.rep + rr - t * pl.rep;
                *reinterpret_cast<float4*>(a.out + ((long long)b * a.T + t) * a.ld_out + h * HD + (i - row * (HD / 4)) * 4) =
                    make_float4(0.f, 0.f, 0.f, 0.f);
            }
            rows = min(RT, sq.n_new * pl.rep - r0);
            if (rows <= 0) return;  // the whole cluster
        } else {
            int len = kvq_len(sq);
            while (gpos >= base + len && b + 1 < a.B) {  // gpos is below the total: a sequence with work follows
                base += len;
                sq = kvq_seq(a, pl, ++b);
                len = kvq_len(sq);
            }
            if (gpos >= base + len) break;
            const int per_unit = sq.blocks + KA_UNIT_COST, unit = (gpos - base) / per_unit;
            ub = base + unit * per_unit;
            blk0 = kvq_cut(gpos - ub, sq.blocks);
            blk1 = min(sq.blocks, range.g1 - ub < per_unit ? kvq_cut(range.g1 - ub, sq.blocks) : per_unit);
            gpos = min(range.g1, ub + per_unit);
            if (blk0 >= blk1) continue;
            const int tiles = sq.units / a.n_kv;
            kvh = unit / tiles;
            tile = unit - kvh * tiles;
            r0 = tile * RT;
            rows = min(RT, sq.n_new * pl.rep - r0);
        }

        // this warp's turns of PB blocks: warp, and every KA_WARPS-th from there
        const int turns = (blk1 - blk0 + F::PB - 1) / F::PB, n_mine = turns > warp ? (turns - warp + KA_WARPS - 1) / KA_WARPS : 0;
        const long long where = sq.slot * a.slot_bytes + kvh * a.head_bytes + (long long)(blk0 + warp * F::PB) * F::BLOCK + lane * 16;
        const uint8_t *kc = a.kc + where, *vc = a.vc + where;
        int left = blk1 - blk0 - warp * F::PB;  // blocks from the next turn on
        uint32_t fill = ring;
        auto fetch = [&]() {  // the next turn into the next stage
            if (left > 0) {
                const uint32_t dst = fill + lane * 16;
                const int bytes = left >= F::PB ? F::PB * F::BLOCK : F::BLOCK;  // (a segment's last turn may lack a block)
                if (F::PB == 1 || left >= F::PB) {
#pragma unroll
                    for (int c = 0; c < F::PB * F::BLOCK; c += 512)
                        if (c + 512 <= F::PB * F::BLOCK || lane * 16 < F::PB * F::BLOCK - c) {
                            ka_copy16(dst + c, kc + c);
                            ka_copy16(dst + F::PB * F::BLOCK + c, vc + c);
                        }
                } else {
                    for (int c = 0; c + lane * 16 < bytes; c += 512) {
                        ka_copy16(dst + c, kc + c);
                        ka_copy16(dst + F::PB * F::BLOCK + c, vc + c);
                    }
                }
                left -= KA_WARPS * F::PB;
                kc += KA_WARPS * F::PB * F::BLOCK;
                vc += KA_WARPS * F::PB * F::BLOCK;
                fill = fill == ring + (F::ST - 1) * F::STAGE ? ring : fill + F::STAGE;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < F::ST - 1; ++i) fetch();

        // q as A fragments in shared memory.  Rows g and g + 8 of M: the tile's rows (MODE 2), or the high and the low
        // half of one.  Each warp lays out every KA_WARPS-th group.
        constexpr int NQ = (NG + KA_WARPS - 1) / KA_WARPS;
        float fr[NR];  // out of q's scale, to powers of two
        int lim[NR];   // last position that the row sees
        {
            float x[NR][NQ][8];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                const int row = MODE == 0 ? g & 3 : nr * 8 + g, rr = r0 + row;
                const bool valid = row < rows;
                const int t = valid ? rr / pl.rep : 0, h = valid ? kvh * pl.rep + rr - t * pl.rep : 0;
                const float* qp = a.q + ((long long)b * a.T + t) * a.ld_q + h * HD + tq * 8;
                float mx = 0.f;
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    const int k = i * KA_WARPS + warp;
                    const bool in = valid && k < NG;
                    const float4 u = in ? *reinterpret_cast<const float4*>(qp + k * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
                    const float4 v = in ? *reinterpret_cast<const float4*>(qp + k * 32 + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
                    float* y = x[nr][i];
                    y[0] = u.x; y[1] = u.y; y[2] = u.z; y[3] = u.w;
                    y[4] = v.x; y[5] = v.y; y[6] = v.z; y[7] = v.w;
#pragma unroll
                    for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(y[j]));
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
                if (tq == 0 && row < RT) q_max[warp * RT + row] = mx;
                lim[nr] = sq.n_ctx + (r0 + row) / pl.rep;
            }
            __syncthreads();
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                const int row = MODE == 0 ? g & 3 : nr * 8 + g;
                float mx = q_max[row];
#pragma unroll
                for (int i = 1; i < KA_WARPS; ++i) mx = fmaxf(mx, q_max[i * RT + row]);
                // the row's largest value goes to [2^13, 2^14); rows of zeros, subnormals and infinities as they are
                const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
                const int sh = ex <= -127 || ex == 128 ? 0 : max(-120, min(120, 13 - ex));
                const float sc = __int_as_float((sh + 127) << 23);
                fr[nr] = __int_as_float((127 - sh) << 23) * log2e_d;
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    const int k = i * KA_WARPS + warp;
                    if (k >= NG) continue;
                    uint32_t* dst = reinterpret_cast<uint32_t*>(qs + k * 1024 + lane * 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        // codes 4 apart share a register in 4 bits (odd ones times 16), codes 2 apart in 8
                        const int e0 = BITS == 4 ? j : (j >> 1) * 4 + (j & 1), e1 = BITS == 4 ? j + 4 : e0 + 2;
                        const float down = BITS == 4 && (j & 1) ? sc * 0.0625f : sc;
                        const float u = x[nr][i][e0] * down, v = x[nr][i][e1] * down;
                        const uint32_t hi = ka_pack(u, v);
                        const float2 f = ka_unpack(hi);
                        const uint32_t lo = ka_pack(u - f.x, v - f.y);
                        uint32_t* d = dst + (j >> 1) * 128 + (j & 1) * 2;
                        if (MODE == 2) {
                            d[nr] = hi;
                            d[NG * 256 + nr] = lo;
                        } else {
                            d[0] = hi;
                            d[1] = lo;
                        }
                    }
                }
            }
            __syncthreads();
        }
        const int open_to = sq.n_ctx + r0 / pl.rep;  // every row sees the positions up to here

        // Columns 2 tq and 2 tq + 1 of the output; dims 16 d + 2 g and one on.
        float o[NR][HD / 16][4];
        // Row g (and g + 8): largest score and the one that moves it (both in q's scale), exponent that p is
        // relative to, sum
        float m[NR], ref[NR], thr[NR], l[NR];
        uint32_t top[NR];          // largest V scale that the row saw, rounded up within its binary order
        uint32_t top_all = 0;      // the least of all rows' tops, twice
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) o[nr][j][0] = o[nr][j][1] = o[nr][j][2] = o[nr][j][3] = 0.f;
            m[nr] = thr[nr] = -INFINITY;
            ref[nr] = l[nr] = 0.f;
            top[nr] = 0;
        }

        // One turn at `at` (its K, then its V), from position p0 on.
        constexpr int PB = F::PB;
        auto turn = [&](auto masked_c, const uint8_t* at, const int p0) {
            constexpr bool MASKED = decltype(masked_c)::value;
            const int end = MASKED ? min(p0 + 16 * PB, blk1 * 16) : 0;
            // scores of row g (and g + 8) against positions 2 tq, 2 tq + 1 (x, y), and 8 on, of each block
            float2 x[PB][NR][2];
#pragma unroll
            for (int pb = 0; pb < PB; ++pb) {
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) x[pb][nr][0] = x[pb][nr][1] = make_float2(0.f, 0.f);
                const uint8_t* kb = at + pb * F::BLOCK;
                uint32_t w[W], s[2 * NG];
                ka_words<W>(kb, lane, w);
                ka_scales<NG>(kb + CODES, tq, s);
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    uint32_t qf[QP][2][4];
#pragma unroll
                    for (int part = 0; part < QP; ++part) {
                        ka_lds4(q_at + (part * NG + k) * 1024, qf[part][0]);
                        ka_lds4(q_at + (part * NG + k) * 1024 + 512, qf[part][1]);
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t f[4];
                        if (BITS == 4) {
                            ka_nibbles(w[half * (W / 2) + k], magic, f);
                        } else {
                            ka_bytes(w[half * (W / 2) + 2 * k], magic, f[0], f[1]);
                            ka_bytes(w[half * (W / 2) + 2 * k + 1], magic, f[2], f[3]);
                        }
                        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int part = QP - 1; part >= 0; --part) {  // the low halves first
                            ka_mma(c, qf[part][0], f[0], f[1]);
                            ka_mma(c, qf[part][1], f[2], f[3]);
                        }
                        const float2 sc = make_float2(ka_scale(s, half * 2, k), ka_scale(s, half * 2 + 1, k));
                        x[pb][NR - 1][half] = ka_fma2(make_float2(c[2], c[3]), sc, x[pb][NR - 1][half]);
                        x[pb][0][half] = ka_fma2(make_float2(c[0], c[1]), sc, x[pb][0][half]);
                    }
                }
            }
            const uint8_t* vb = at + PB * F::BLOCK;
            auto seen = [&](int pb, int nr, int e) {
                const int pos = p0 + 16 * pb + 2 * tq + (e & 1) + (e >> 1) * 8;
                return !MASKED || (pos <= lim[nr] && pos < end);
            };
            bool raise = false;
#pragma unroll
            for (int pb = 0; pb < PB; ++pb) {
                // a lane looks at one word of V's scales
                const uint32_t word = *reinterpret_cast<const uint32_t*>(vb + pb * F::BLOCK + CODES + min(lane, HD / 4 - 1) * 4) & 0x7FFF7FFFu;
                raise |= (word & 0xFFFFu) > top_all || word >> 16 > top_all;
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (!seen(pb, nr, 2 * e)) x[pb][nr][e].x = -INFINITY;
                        if (!seen(pb, nr, 2 * e + 1)) x[pb][nr][e].y = -INFINITY;
                        raise |= x[pb][nr][e].x > thr[nr] || x[pb][nr][e].y > thr[nr];
                    }
            }
            if (__any_sync(0xFFFFFFFFu, raise)) {
                uint32_t least = 0xFFFFu;
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    float mx = m[nr];
                    uint32_t tp = top[nr];
#pragma unroll
                    for (int pb = 0; pb < PB; ++pb) {
                        uint32_t vs[2 * NG];
                        ka_scales<NG>(vb + pb * F::BLOCK + CODES, tq, vs);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            mx = fmaxf(mx, e & 1 ? x[pb][nr][e >> 1].y : x[pb][nr][e >> 1].x);
                            if (seen(pb, nr, e)) {
#pragma unroll
                                for (int k = 0; k < NG; ++k) {  // NaN and infinity have no say
                                    const uint32_t v = __half_as_ushort(__float2half_rn(fabsf(ka_scale(vs, e, k))));
                                    if (v < 0x7C00u) tp = max(tp, v);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int s = 1; s < 4; s <<= 1) {
                        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, s));
                        tp = max(tp, __shfl_xor_sync(0xFFFFFFFFu, tp, s));
                    }
                    // a row moves by what it sees alone, whichever row asked
                    float f = 1.0f;
                    if (mx > thr[nr] || tp > top[nr]) {
                        tp |= 0x3FFu;  // scales are below 2^(tp / 1024 - 14)
                        const float nref = mx == -INFINITY ? 0.f : mx * fr[nr] - (float)(15 - KA_SLACK + 14 - (int)(tp >> 10));
                        // (a row that saw nothing yet has sums of zero, or NaN, which stays)
                        f = m[nr] == -INFINITY ? 0.f : ka_exp2(ref[nr] - nref);
                        m[nr] = mx;
                        thr[nr] = mx + (float)KA_SLACK / fr[nr];
                        ref[nr] = nref;
                        top[nr] = tp;
                        l[nr] *= f;
                    }
                    least = min(least, top[nr]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float fc = __shfl_sync(0xFFFFFFFFu, f, (2 * tq + j) * 4);
#pragma unroll
                        for (int d = 0; d < HD / 16; ++d) {
                            o[nr][d][j] *= fc;
                            o[nr][d][2 + j] *= fc;
                        }
                    }
                }
                top_all = __reduce_min_sync(0xFFFFFFFFu, least);
            }
#pragma unroll
            for (int pb = 0; pb < PB; ++pb) {
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float2 y = ka_fma2(x[pb][nr][e], make_float2(fr[nr], fr[nr]), make_float2(-ref[nr], -ref[nr]));
                        x[pb][nr][e] = make_float2(ka_exp2(y.x), ka_exp2(y.y));
                        l[nr] += x[pb][nr][e].x + x[pb][nr][e].y;
                    }
                uint32_t w[W], vs[2 * NG];
                ka_scales<NG>(vb + pb * F::BLOCK + CODES, tq, vs);
                ka_words<W>(vb + pb * F::BLOCK, lane, w);
                // p is cut after 11 bits, and what is left again; MODE 0: columns 0 .. 3 take the first part, 4 .. 7 the
                // second (the cut of the others is to nothing)
                const uint32_t cut = MODE == 0 && g < 4 ? 0u : 0xFFFFE000u;
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    uint32_t pf[NR][PP][2];
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            float2 y = ka_mul2(x[pb][nr][half], make_float2(ka_scale(vs, 2 * half, k), ka_scale(vs, 2 * half + 1, k)));
                            if (MASKED) {  // an unseen position's scale may be NaN
                                if (!seen(pb, nr, 2 * half)) y.x = 0.f;
                                if (!seen(pb, nr, 2 * half + 1)) y.y = 0.f;
                            }
                            const float2 h = make_float2(__uint_as_float(__float_as_uint(y.x) & cut), __uint_as_float(__float_as_uint(y.y) & cut));
                            const float2 z = ka_fma2(h, make_float2(-1.f, -1.f), y);
                            if (MODE != 0) pf[nr][0][half] = ka_pack_rz(y.x, y.y);
                            pf[nr][PP - 1][half] = ka_pack_rz(z.x, z.y);
                        }
#pragma unroll
                    for (int d = 2 * k; d < 2 * k + 2; ++d) {
                        uint32_t v[4];
                        if (BITS == 4) {
                            ka_nibbles(w[d], magic, v);
                        } else {
                            ka_bytes(w[2 * d], magic, v[0], v[2]);
                            ka_bytes(w[2 * d + 1], magic, v[1], v[3]);
                        }
#pragma unroll
                        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                            for (int part = PP - 1; part >= 0; --part) ka_mma(o[nr][d], v, pf[nr][part][0], pf[nr][part][1]);
                    }
                }
            }
        };

        uint32_t at = ring_at;
        int p0 = (blk0 + warp * PB) * 16;
        const int last = min(open_to, blk1 * 16 - 1);  // up to here every position of a turn is seen
#pragma unroll 1
        for (int i = 0; i < n_mine; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(F::ST - 2) : "memory");
            __syncwarp();  // everyone's copies of this stage are visible, and the stage before is read
            fetch();
            if (p0 + 16 * PB - 1 <= last) turn(std::false_type(), smem + at, p0);
            else turn(std::true_type(), smem + at, p0);
            p0 += KA_WARPS * PB * 16;
            at = at == ring_at + (F::ST - 1) * F::STAGE ? ring_at : at + F::STAGE;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        __syncthreads();
        // the warp's rows into its slot: dims 16 d + 2 g and one on, rows 2 tq and one on
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = nr * 8 + 2 * tq + j;
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) {
                    float2 y = make_float2(o[nr][d][j], o[nr][d][2 + j] * (BITS == 4 ? 0.0625f : 1.0f));
                    if (MODE == 0) {
                        y.x += __shfl_xor_sync(0xFFFFFFFFu, y.x, 2);
                        y.y += __shfl_xor_sync(0xFFFFFFFFu, y.y, 2);
                    }
                    if (row < RT) *reinterpret_cast<float2*>(slot_all + (warp * RT + row) * HD + 16 * d + 2 * g) = y;
                }
            }
            l[nr] += __shfl_xor_sync(0xFFFFFFFFu, l[nr], 1);
            l[nr] += __shfl_xor_sync(0xFFFFFFFFu, l[nr], 2);
            const int row = nr * 8 + g;
            if (tq == 0 && row < RT) {
                // a warp without blocks, or whose rows saw nothing: its exponent says so
                const bool none = n_mine == 0 || (m[nr] == -INFINITY && l[nr] == 0.f);
                stat[warp * RT + row] = none ? -INFINITY : ref[nr];
                stat[(KA_WARPS + warp) * RT + row] = l[nr];
            }
        }
        __syncthreads();
        const bool begins = blk0 == 0, ends = blk1 == sq.blocks, whole = CLUSTER ? pl.split == 1 : begins && ends;
        // what this CTA hands on: rows, then their exponents and sums (CLUSTER: in shared memory, where q was)
        float* part = CLUSTER ? reinterpret_cast<float*>(qs) : parts + (blockIdx.x * 2 + (begins ? 1 : 0)) * kvq_part_floats(RT, HD);
        float* part_stat = CLUSTER ? q_max : part + RT * HD;
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
            if (whole) {
                const int rr = r0 + row, t = rr / pl.rep, h = kvh * pl.rep + rr - t * pl.rep;
                const float inv = L == 0.f ? 0.f : 1.0f / L;
                *reinterpret_cast<float4*>(a.out + ((long long)b * a.T + t) * a.ld_out + h * HD + d) =
                    make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
            } else {
                *reinterpret_cast<float4*>(part + row * HD + d) = y;
                if (d == 0) {
                    part_stat[row] = mx;
                    part_stat[RT + row] = L;
                }
            }
        }
        if (CLUSTER) {
            if (whole) return;
            ka_cluster_sync();
            for (int i = rank * KA_THREADS + threadIdx.x; i < rows * (HD / 4); i += pl.split * KA_THREADS) {
                const int row = i / (HD / 4), d = (i - row * (HD / 4)) * 4;
                float e[KA_MAX_SPLIT], l1[KA_MAX_SPLIT], mx = -INFINITY, L = 0.f;
                float4 u[KA_MAX_SPLIT], y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int c = 0; c < KA_MAX_SPLIT; ++c)
                    if (c < pl.split) {
                        e[c] = ka_remote1(part_stat + row, c);
                        l1[c] = ka_remote1(part_stat + RT + row, c);
                        u[c] = ka_remote4(part + row * HD + d, c);
                    }
#pragma unroll
                for (int c = 0; c < KA_MAX_SPLIT; ++c)
                    if (c < pl.split) mx = fmaxf(mx, e[c]);
#pragma unroll
                for (int c = 0; c < KA_MAX_SPLIT; ++c)
                    if (c < pl.split && e[c] != -INFINITY) {
                        const float f = ka_exp2(e[c] - mx);
                        L = fmaf(l1[c], f, L);
                        y.x = fmaf(u[c].x, f, y.x);
                        y.y = fmaf(u[c].y, f, y.y);
                        y.z = fmaf(u[c].z, f, y.z);
                        y.w = fmaf(u[c].w, f, y.w);
                    }
                const int rr = r0 + row, t = rr / pl.rep, h = kvh * pl.rep + rr - t * pl.rep;
                const float inv = L == 0.f ? 0.f : 1.0f / L;
                *reinterpret_cast<float4*>(a.out + ((long long)b * a.T + t) * a.ld_out + h * HD + d) =
                    make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
            }
            ka_cluster_sync();  // no CTA leaves while another reads its shared memory
            return;
        }
        __syncthreads();
        if (begins) {
            const int last = (ub + sq.blocks - 1) / range.per;  // the CTA with the last block, if its cut stays
            const int c1 = kvq_cut(last * range.per - ub, sq.blocks) >= sq.blocks ? last - 1 : last;
            const KvqDesc de = {ends ? -1 : b, kvh, tile, rows, (int)blockIdx.x, c1};
            if (!ends) open = de;
            if (pl.by_unit && threadIdx.x == 0) desc[(b * a.n_kv + kvh) * pl.tiles + tile] = de;
        }
    }
    if (!pl.by_unit && threadIdx.x == 0) desc[blockIdx.x] = open;

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
// Block (x, y): descriptor x, rows y ROWS on; WAYS warps per row share its parts, a lane per part for the weights
// and per four dims for the sums, eight parts' rows in flight.
template <int ROWS, int WAYS>
__global__ void __launch_bounds__(ROWS * WAYS * 32) tf_kvq_combine_kernel(const KvqAttnArgs a, const KvqPlan pl) {
    __shared__ float4 sum[ROWS][WAYS][32];
    __shared__ float2 stat[ROWS][WAYS];
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lr = warp / WAYS, way = warp % WAYS, r = blockIdx.y * ROWS + lr;
    if (pl.by_unit) {  // a unit that does not exist has no descriptor
        const KvqSeq sq = kvq_seq(a, pl, blockIdx.x / (a.n_kv * pl.tiles));
        if ((int)(blockIdx.x % pl.tiles) * a.n_kv >= sq.units) return;
    }
    const KvqDesc de = static_cast<const KvqDesc*>(a.ws)[blockIdx.x];
    if (de.b < 0 || (int)blockIdx.y * ROWS >= de.rows) return;
    const float* parts = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.ws) + KA_DESC_BYTES);
    const int hd = a.hd, rt = pl.rt, n = de.c1 - de.c0 + 1, d = lane * 4;
    const size_t pf = kvq_part_floats(rt, hd);
    auto part = [&](int i) { return parts + ((size_t)(de.c0 + i) * 2 + (i == 0 ? 1 : 0)) * pf; };
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    // this warp's parts: way, way + WAYS, ...; 32 of them at a time
    const int mine = r < de.rows ? (n - way + WAYS - 1) / WAYS : 0;
#pragma unroll 1
    for (int i0 = 0; i0 < mine; i0 += 32) {
        const int k = min(32, mine - i0);
        auto at = [&](int i) { return part((i0 + i) * WAYS + way); };
        float m = -INFINITY, l = 0.f;
        if (lane < k) {
            const float* p = at(lane) + (size_t)rt * hd + r;
            m = p[0];
            l = p[rt];
        }
        float w = 0.f;
#pragma unroll 1
        for (int i = 0; i < k; i += 8) {
            float4 x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = i + j < k && d < hd ? *reinterpret_cast<const float4*>(at(i + j) + (size_t)r * hd + d)
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
            if (i == 0) {
                const float mx = fmaxf(M, warp_max(m)), to = mx == -INFINITY ? 0.f : mx, alpha = ka_exp2(M - to);
                w = m == -INFINITY ? 0.f : ka_exp2(m - to);
                M = mx;
                L = fmaf(L, alpha, warp_sum(m == -INFINITY ? 0.f : l * w));
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
    if (WAYS > 1) {
        sum[lr][way][lane] = o;
        if (lane == 0) stat[lr][way] = make_float2(M, L);
        __syncthreads();
        if (way != 0) return;
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < WAYS; ++i) mx = fmaxf(mx, stat[lr][i].x);
        L = 0.f;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < WAYS; ++i) {
            if (stat[lr][i].x == -INFINITY) continue;
            const float f = ka_exp2(stat[lr][i].x - mx);
            const float4 u = sum[lr][i][lane];
            L = fmaf(stat[lr][i].y, f, L);
            o.x = fmaf(u.x, f, o.x);
            o.y = fmaf(u.y, f, o.y);
            o.z = fmaf(u.z, f, o.z);
            o.w = fmaf(u.w, f, o.w);
        }
    }
    if (r >= de.rows || d >= hd) return;
    const int rep = pl.rep, rr = de.tile * rt + r, t = rr / rep, h = de.kvh * rep + rr - t * rep;
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    *reinterpret_cast<float4*>(a.out + ((long long)de.b * a.T + t) * a.ld_out + h * hd + d) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// ---- host ------------------------------------------------------------------------------------------
static int kvq_sms() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms < 1 ? 1 : (4 * sms > KA_MAX_GRID ? KA_MAX_GRID / 4 : sms);
}
// CTAs per unit where a cluster takes each unit: as many as leave all units resident, while a warp has no more than
// KA_TURNS blocks at the cache's capacity (lengths are on the device; longer ones are balanced better by ranges).
constexpr int KA_TURNS = 10;
static int kvq_split_of(long long units, int cap, int slots) {
    for (int s = KA_MAX_SPLIT; s >= 1; s >>= 1)
        if (units * s <= slots) return cap / 16 <= s * KA_WARPS * KA_TURNS ? s : 0;
    return 0;
}
static int kvq_mode(int rows) { return rows <= 4 ? 0 : rows <= 8 ? 1 : 2; }

size_t kvq_attn_ws_bytes(int T, int n_head, int n_kv, int hd) {
    const int mode = kvq_mode(T * (n_head / n_kv));
    return KA_DESC_BYTES + (size_t)kvq_sms() * kvq_ctas(mode) * 2 * kvq_part_floats(kvq_rt(mode), hd) * sizeof(float);
}

// Units of 4 rows or more, blocks of 16 positions and a unit's cost.
bool kvq_attn_fits(int B, int T, int n_head, int n_kv, int cap) {
    const int rows = T * (n_head / n_kv), rt = kvq_rt(kvq_mode(rows));
    return (double)B * n_kv * ((rows + rt - 1) / rt) * ((double)cap / 16 + KA_UNIT_COST) < 2147483648.0;
}

static cudaError_t kvq_launch(const void* fn, dim3 grid, int threads, size_t smem, int cluster, void** args, cudaStream_t st, bool pdl) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

template <int BITS, int HD, int MODE, bool CLUSTER>
static cudaError_t kvq_ready() {  // set once per device; twice is harmless
    const void* fn = (const void*)tf_kvq_attn_kernel<BITS, HD, MODE, CLUSTER>;
    static std::atomic<bool> ready[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (ready[dev]) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, KvqCfg<BITS, HD, MODE>::SMEM);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    ready[dev].store(true);
    return cudaSuccess;
}

template <int BITS, int HD, int MODE>
static cudaError_t mode_launch(const KvqAttnArgs& a, cudaStream_t st) {
    using F = KvqCfg<BITS, HD, MODE>;
    KvqPlan pl;
    const int slots = kvq_sms() * F::CTAS;
    pl.rt = F::RT;
    pl.rep = a.n_head / a.n_kv;
    pl.tiles = (a.T * pl.rep + F::RT - 1) / F::RT;
    const long long units = (long long)a.B * a.n_kv * pl.tiles;
    pl.by_unit = units <= slots;
    pl.split = kvq_split_of(units, a.cap, slots);
    KvqAttnArgs aa = a;
    void* args[] = {&aa, &pl};
    if (pl.split) {
        pl.grid = (int)units * pl.split;
        const cudaError_t e = kvq_ready<BITS, HD, MODE, true>();
        if (e != cudaSuccess) return e;
        return kvq_launch((const void*)tf_kvq_attn_kernel<BITS, HD, MODE, true>, dim3(pl.grid), KA_THREADS, F::SMEM, pl.split, args, st, false);
    }
    pl.grid = slots;
    cudaError_t e = kvq_ready<BITS, HD, MODE, false>();
    if (e != cudaSuccess) return e;
    e = kvq_launch((const void*)tf_kvq_attn_kernel<BITS, HD, MODE, false>, dim3(pl.grid), KA_THREADS, F::SMEM, 1, args, st, false);
    if (e != cudaSuccess) return e;
    const int found = pl.by_unit ? (int)units : pl.grid;
    // few units have many parts each: eight warps to a row
    if (found * F::RT <= 1024) return kvq_launch((const void*)tf_kvq_combine_kernel<1, 8>, dim3(found, F::RT), 256, 0, 1, args, st, true);
    return kvq_launch((const void*)tf_kvq_combine_kernel<4, 1>, dim3(found, F::RT / 4), 128, 0, 1, args, st, true);
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
