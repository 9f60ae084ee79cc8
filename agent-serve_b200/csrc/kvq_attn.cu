// Attention over a quantised KV cache (Q4_0 / Q8_0, layout in kvq.cuh): T new rows per sequence, row t of
// sequence b seeing cache rows 0 .. n_ctx[b] + t; T = 1 is decode.
//
// Row (b, t, h): s_j = q . k_j / sqrt(hd), p_j = exp(s_j - max s), out = sum p_j v_j / sum p_j.
//
// Bound by the cache's bytes, then by instructions: a position of one kv head is 2 hd codes (144 bytes with its scales
// for 128 dims in 4 bits), and at 6.5 TB/s an SM has 6.2 cycles for those, 25 issue slots.  Hence mma.sync m16n8k16
// with the codes in the order of its fragments: a 32-bit word of eight codes is a shift, four LOP3 and four HADD2 away
// from four operand registers, and no shared-memory pass is needed.  tcgen05 would want the codes unpacked through
// shared memory, and 64 rows or more.  The output has the dims as M and the rows as N (V transposed is the A operand).
// The scores, by the rows of a kv head (times the new rows):
//   up to 4 (FewRows)   positions as M, rows as N: the 8 columns hold the high and the low half of q, and of p, side by
//                       side; probabilities go to the second product's operand by movmatrix;
//   more (ManyRows)     rows as M, positions as N: the scores' registers are the second product's operand as they
//                       stand; up to 8 rows, the 16 rows of M hold q's two halves.
// 64 sequences over 8192 positions, 8 kv heads of 128, 4 rows each, 4 bits: 148 us as FewRows, 191 as ManyRows; 16 sequences
// of 16 new rows over up to 4000 positions, 64 dims: 104 and 56.
//
// Arithmetic (fp32-equivalent).  Codes less their zero are exact in f16: (code | 0x6400) is 1024 + code, and
// the high nibble in place 1024 + 16 code; the 16 is taken out of q (K) or of the output row (V).  q is split
// into two f16 halves after a power-of-two scale of its row (22 bits or more).  A group's products are summed from
// zero and enter the score by an fp32 fma with the group's scale.  V's scales multiply p (they differ by group of
// dims, so p is split once for each group): p = 2^(x - m + k), p scale as an f16 and what it leaves, times 2^11, as
// another, both rounded to nearest.  m is the row's running maximum, up to 2^8 behind; k comes from the largest V scale
// that the row has seen, so that p scale stays below 2^15 and the largest is 2^6 at least; the second half keeps 2^-36.
// A group of dims whose values are 2^-18 of the row's largest, or a position whose weight is, so has 24 bits.  (Without
// the 2^11, cut towards zero, 64 sequences over up to 8128 positions take 90.5 us instead of 91.6 and calls with 5 rows or
// more a kv head 1 to 8 % less, but a group at 2^-14 is off by 2e-5 to 4e-5, and 20000 weights of e^-18 by 7e-5.)  k is a
// row's own: its bits must not hang on what only another row sees.  A block's P V is summed from zero and joins the output
// by an fp32 addition (3 % of the time): the matrix accumulator truncates, and a sum of one sign carried in it through
// 166 blocks is off by 2.5e-5.
//
// Work is cut into units (sequence, kv head, row tile) and each unit into blocks of 16 positions.  A CTA's warps take
// its blocks in turn, each with its own ring of cp.async copies (no barrier in the loop), and join at the end.
//   Short caches: a cluster of 1 to 8 CTAs per unit, which join over distributed shared memory: one launch.
//   Else the blocks of all units, in order, are dealt out to the CTAs in equal contiguous ranges (lengths are read on
//   the device, so ragged batches stay balanced); a unit that a range cuts leaves partial results for
//   tf_kvq_combine_kernel.
// All joins are in a fixed order: results repeat bit for bit.
//
// Measured: 64 sequences over 1161 to 8128 positions, 8 kv heads of 128, 4 rows each: 4 bits 92 us (3.7 TB/s: 384
// instructions per block and warp, issue slots 64 to 67 %, FMA pipe 45 %, ALU 42 %, DRAM 40 %, 24 bytes a thread spilled; the
// copies alone take 62 us); 32 such sequences in 8 bits 61 us (5.3 TB/s).  1 sequence over 96 positions, 64 dims: 4.0 us in a cache
// of 112 positions, a launch and four dependent reads; 6.1 in one of 8192, where the capacity asks for ranges.
#include <atomic>
#include <type_traits>

#include "kvq.cuh"

namespace tfb {

constexpr int KA_THREADS = 128;
constexpr int KA_WARPS = KA_THREADS / 32;
// Blocks that a unit's start and end take the time of in a range: 8 / 16 / 24 / 32, 64 sequences over up to 8128 positions
// 93.2 / 91.7 / 92.0 / 92.9 us, 128 over up to 4000 (8 bits, 64 dims) 68.4 / 65.4 / 63.8 / 63.9, 16 of 16 new rows 58.2 /
// 56.6 / 56.5 / 56.8.
constexpr int KA_UNIT_COST = 24;
// Blocks of a CTA's range at least: 8 / 16 / 24 / 32, 1 sequence over 32001 positions 14.3 / 10.7 / 11.0 / 11.4 us, 1 over
// 16000 (64 dims) 11.8 / 11.3 / 10.6 / 11.7, 1 of 4 new rows over 8000 14.8 / 15.7 / 16.0 / 17.9.
constexpr int KA_MIN_RANGE = 24;
constexpr int KA_MAX_SPLIT = 8;    // CTAs of a cluster
// A cut this near to a unit's first or last block moves there: 0 / 6, 1 sequence over 96 positions in a cache of 8192 7.0 / 6.1
// us, 64 over up to 100 8.4 / 7.5, 64 over up to 8128 91.9 / 92.3, 33 of 4 rows over up to 2000 24.7 / 26.1.
constexpr int KA_SNAP = 6;
// Binary orders that a running maximum may lag behind: 4 / 6 / 8, 64 sequences over up to 8128 positions 92.6 / 91.8 / 91.6 us,
// 32 of 5 new rows over 1144 17.0 / 16.4 / 16.3.
constexpr int KA_SLACK = 8;
constexpr int KA_MAX_GRID = 1024;  // descriptors of 32 bytes in the workspace's first 32 KB
constexpr size_t KA_DESC_BYTES = 32768;

struct KvqPlan {
    int grid;
    int rt;        // rows per row tile
    int rep;       // query heads per kv head
    unsigned inv;  // 2^32 / rep, rounded up
    int tiles;     // row tiles of T rows
    int split;     // CTAs of a unit, one cluster; 0: ranges of all units' blocks
    int by_unit;   // descriptors are found by unit (there are at most `grid`), else by the CTA that begins it
};
// x / rep for x < 2^16 and rep <= 1024 (the error x 2^-32 stays below 1 / rep)
__host__ __device__ __forceinline__ int kvq_div(int x, int rep, unsigned inv) {
    return rep == 1 ? x : (int)((unsigned long long)(unsigned)x * inv >> 32);
}
struct alignas(32) KvqDesc {  // a unit split over CTAs c0 .. c1
    int b, kvh, tile, rows, c0, c1;  // b < 0: no unit, or one that was not split
};

__host__ __device__ inline size_t kvq_part_floats(int rt, int hd) { return (size_t)rt * (hd + 2); }

// Row tiles: 0: 4 rows, 1: 8, 2: 16.  (32 share a block's codes over more rows, but need 255 registers at 128 dims.  Before the
// second half of p carried 2^11: 32 sequences of 5 x 6 rows over 1144 positions 16.2 -> 19.3 us, 16 of 16 x 4 over 4000, 64
// dims, 55.9 -> 57.4.)
__host__ __device__ constexpr int kvq_rt(int mode) { return mode == 0 ? 4 : mode == 1 ? 8 : 16; }

// 168 or 128 registers a thread (at 128 dims 48 to 84 and up to 28 bytes spilled)
__host__ __device__ constexpr int kvq_ctas(int mode) { return mode == 2 ? 3 : 4; }

template <int BITS, int HD, int MODE>
struct KvqCfg {
    static constexpr int RT = kvq_rt(MODE);
    static constexpr int CTAS = kvq_ctas(MODE);                    // per SM
    static constexpr int BLOCK = kvq_block_bytes(BITS, HD);
    static constexpr int STAGE = 2 * BLOCK;                        // K, then V, of 16 positions
    static constexpr int SLOT = RT * HD * 4;                       // a warp's output rows
    static constexpr int QF = (MODE == 2 ? 2 : 1) * HD / 32 * (MODE == 0 ? 512 : 1024);  // q's fragments
    static constexpr int QS = QF > SLOT ? QF : SLOT;               // later a CTA's output rows
    static constexpr int STAT = KA_WARPS * RT * 12;
    static constexpr int ROOM = 227 * 1024 / CTAS - 1024 - STAT - QS;
    static constexpr int FIT = ROOM / (KA_WARPS * STAGE);
    static constexpr int ST = FIT > 8 ? 8 : FIT;                   // stages of a warp's ring
    static constexpr int RING = ST * STAGE > SLOT ? ST * STAGE : SLOT;  // output rows take the rings' place
    static constexpr int SMEM = KA_WARPS * RING + STAT + QS;
    static_assert(ST >= 2 && SMEM <= 227 * 1024 / CTAS - 1024, "two stages at least");
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
// 8 x 8 halves, row g in the lanes 4 g .. 4 g + 3, to their transpose
__device__ __forceinline__ uint32_t ka_trans(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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
__device__ __forceinline__ void ka_add4(float (&a)[4], const float (&b)[4]) {
    asm("{\n\t.reg .b64 a0, a1, b0, b1;\n\t"
        "mov.b64 a0, {%0, %1};\n\tmov.b64 a1, {%2, %3};\n\tmov.b64 b0, {%4, %5};\n\tmov.b64 b1, {%6, %7};\n\t"
        "add.rn.f32x2 a0, a0, b0;\n\tadd.rn.f32x2 a1, a1, b1;\n\t"
        "mov.b64 {%0, %1}, a0;\n\tmov.b64 {%2, %3}, a1;\n\t}"
        : "+f"(a[0]), "+f"(a[1]), "+f"(a[2]), "+f"(a[3])
        : "f"(b[0]), "f"(b[1]), "f"(b[2]), "f"(b[3]));
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
// the scales of positions g and g + 8: NG = HD / 32 groups each, two to a word
template <int NG>
__device__ __forceinline__ void ka_scales(const uint8_t* p, int g, uint32_t (&s)[NG]) {
    const uint8_t* q = p + g * (4 * NG);
    if (NG % 4 == 0) {
        ka_lds4(q, s);
    } else if (NG % 2 == 0) {
        ka_lds2(q, s);
    } else {
#pragma unroll
        for (int i = 0; i < NG; ++i) s[i] = *reinterpret_cast<const uint32_t*>(q + 4 * i);
    }
}
// Scale of group k of position g + 8 half.
template <int NG>
__device__ __forceinline__ float ka_scale(const uint32_t (&s)[NG], int half, int k) {
    const int i = half * NG + k;
    const __half2 h = *reinterpret_cast<const __half2*>(&s[i >> 1]);
    return i & 1 ? __high2float(h) : __low2float(h);
}

// ---- the split of the blocks over the CTAs ------------------------------------------------------------
struct KvqSeq {
    int slot, n_ctx, n_new, blocks, units;
    bool bad;
};
__device__ __forceinline__ KvqSeq kvq_seq(const KvqAttnArgs& a, int rep, int rt, int b) {
    KvqSeq s;
    s.slot = a.slots ? a.slots[b] : b;
    s.n_ctx = a.n_ctx[b];
    s.n_new = a.n_new ? a.n_new[b] : a.T;
    // without new rows a sequence is empty (a padded batch), whatever its slot and length say
    s.bad = s.n_new < 0 || s.n_new > a.T || (s.n_new > 0 && (s.slot < 0 || s.slot >= a.n_slots || s.n_ctx < 0 || s.n_ctx > a.cap - s.n_new));
    if (s.bad) s.n_new = 0;
    s.blocks = s.n_new ? (s.n_ctx + s.n_new + 15) >> 4 : 0;
    s.units = a.n_kv * ((s.n_new * rep + rt - 1) / rt);
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
template <int RT>
__device__ __forceinline__ KvqRange kvq_range(const KvqAttnArgs& a, const KvqPlan& pl) {
    const int lane = threadIdx.x & 31;
    const int chunk = (a.B + 31) >> 5, lo = min(a.B, lane * chunk), hi = min(a.B, lo + chunk);
    int mine = 0;
#pragma unroll 4
    for (int b = lo; b < hi; ++b) {
        const KvqSeq s = kvq_seq(a, pl.rep, RT, b);
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

// ---- a warp's work on a unit's blocks --------------------------------------------------------------------
// What a segment of a unit is to its warps.
struct KvqSeg {
    int b, kvh, r0, rows;  // rows r0 .. r0 + rows - 1 of the unit's (new row, head) pairs
    int rep, T, n_ctx;
    unsigned inv;
    int open_to;           // every row sees the positions up to here
};
__device__ __forceinline__ const float* kvq_query(const KvqAttnArgs& a, const KvqSeg& sg, int row, int hd) {
    const int rr = sg.r0 + row, t = kvq_div(rr, sg.rep, sg.inv), h = sg.kvh * sg.rep + rr - t * sg.rep;
    return a.q + ((long long)sg.b * sg.T + t) * a.ld_q + h * hd;
}
// A row's largest value goes to [2^13, 2^14); rows of zeros, subnormals and infinities stay as they are.
__device__ __forceinline__ int kvq_shift(float mx) {
    const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
    return ex <= -127 || ex == 128 ? 0 : max(-120, min(120, 13 - ex));
}
template <int RT>
__device__ __forceinline__ float kvq_row_max(const float* q_max, int row) {  // over the warps' groups
    float mx = q_max[row];
#pragma unroll
    for (int i = 1; i < KA_WARPS; ++i) mx = fmaxf(mx, q_max[i * RT + row]);
    return mx;
}
// Eight dims of q from 8 tq on of group k, as f16 halves in the order of a word's codes: registers 0 .. 3 pair codes 4
// apart in 4 bits (odd ones times 16), 2 apart in 8.
template <int BITS>
__device__ __forceinline__ void kvq_split_q(const float (&x)[8], float sc, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e0 = BITS == 4 ? j : (j >> 1) * 4 + (j & 1), e1 = BITS == 4 ? j + 4 : e0 + 2;
        const float down = BITS == 4 && (j & 1) ? sc * 0.0625f : sc;
        const float u = x[e0] * down, v = x[e1] * down;
        hi[j] = ka_pack(u, v);
        const float2 f = ka_unpack(hi[j]);
        lo[j] = ka_pack(u - f.x, v - f.y);
    }
}
// A row's running state: largest score and the one that moves it (both in q's scale), minus the exponent that p is
// relative to, sum, and the largest V scale that the row saw, rounded up within its binary order.
struct KvqRow {
    float m, thr, nref, l;
    uint32_t top;
    __device__ __forceinline__ void clear() {
        m = thr = -INFINITY;
        nref = l = 0.f;
        top = 0;
    }
    // New largest score and V scale; returns what the row's sums are multiplied with.  A row moves by what it sees
    // alone, whichever row asked.
    __device__ __forceinline__ float move(float mx, uint32_t tp, float fr) {
        if (!(mx > thr || tp > top)) return 1.0f;
        tp |= 0x3FFu;  // scales are below 2^(tp / 1024 - 14)
        const float r = mx == -INFINITY ? 0.f : (float)(15 - KA_SLACK + 14 - (int)(tp >> 10)) - mx * fr;
        const float f = m == -INFINITY ? 0.f : ka_exp2(r - nref);  // (nothing seen yet: sums of zero, or NaN, which stays)
        m = mx;
        thr = mx + (float)KA_SLACK / fr;
        nref = r;
        top = tp;
        l *= f;
        return f;
    }
    __device__ __forceinline__ bool none() const { return m == -INFINITY && l == 0.f; }
};
__device__ __forceinline__ uint32_t ka_scale_bits(uint32_t v, uint32_t top) {  // NaN and infinity have no say
    v &= 0x7FFFu;
    return v < 0x7C00u ? max(v, top) : top;
}
// Whether a V scale of a block is above `top` (a lane looks at one word of them).
template <int HD>
__device__ __forceinline__ bool ka_scale_above(const uint8_t* scales, int lane, uint32_t top) {
    const uint32_t word = *reinterpret_cast<const uint32_t*>(scales + min(lane, HD / 4 - 1) * 4) & 0x7FFF7FFFu;
    return (word & 0xFFFFu) > top || word >> 16 > top;
}
__device__ __forceinline__ uint32_t ka_magic() {
    uint32_t m;
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(m));
    return m;
}

// Up to 4 rows.  Column c of N is row c & 3: the high half below 4, the low half from 4 on.  A thread holds
// columns 2 tq and 2 tq + 1, positions g and g + 8 of a block, and dims 16 d + 2 g and one on of the output.
template <int BITS, int HD>
struct FewRows {
    static constexpr int RT = 4, NG = HD / 32, W = HD * BITS / 64, CODES = kvq_code_bytes(BITS, HD), BLOCK = kvq_block_bytes(BITS, HD);
    static constexpr int NQ = (NG + KA_WARPS - 1) / KA_WARPS;
    const uint8_t* q_at;
    int lane, g, tq;
    uint32_t magic;
    float2 fr;  // out of q's scale, to powers of two
    int2 lim;   // last position that the row sees
    KvqRow r0, r1;
    float o[HD / 16][4];
    uint32_t top_all;  // the least of all rows' tops

    // q to [NG][lane] four registers; each warp lays out every KA_WARPS-th group.
    __device__ __forceinline__ void load_q(const KvqAttnArgs& a, const KvqSeg& sg, uint8_t* qs, float* q_max, int warp, float log2e_d) {
        lane = threadIdx.x & 31;
        g = lane >> 2;
        tq = lane & 3;
        magic = ka_magic();
        q_at = qs + lane * 16;
        float x[NQ][8], mx = 0.f;
        const bool valid = (g & 3) < sg.rows;
        const float* qp = kvq_query(a, sg, valid ? g & 3 : 0, HD) + tq * 8;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int k = i * KA_WARPS + warp;
            const bool in = valid && k < NG;
            const float4 u = in ? *reinterpret_cast<const float4*>(qp + k * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
            const float4 v = in ? *reinterpret_cast<const float4*>(qp + k * 32 + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            float* y = x[i];
            y[0] = u.x; y[1] = u.y; y[2] = u.z; y[3] = u.w;
            y[4] = v.x; y[5] = v.y; y[6] = v.z; y[7] = v.w;
#pragma unroll
            for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(y[j]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
        if (tq == 0 && g < RT) q_max[warp * RT + g] = mx;
        __syncthreads();
        const float sc = __int_as_float((kvq_shift(kvq_row_max<RT>(q_max, g & 3)) + 127) << 23);
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int k = i * KA_WARPS + warp;
            if (k >= NG) continue;
            uint32_t hi[4], lo[4];
            kvq_split_q<BITS>(x[i], sc, hi, lo);
            *reinterpret_cast<uint4*>(qs + k * 512 + lane * 16) =
                g < 4 ? make_uint4(hi[0], hi[1], hi[2], hi[3]) : make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        const int c = (2 * tq) & 3;
        fr.x = __int_as_float((127 - kvq_shift(kvq_row_max<RT>(q_max, c))) << 23) * log2e_d;
        fr.y = __int_as_float((127 - kvq_shift(kvq_row_max<RT>(q_max, c + 1))) << 23) * log2e_d;
        lim.x = sg.n_ctx + kvq_div(sg.r0 + c, sg.rep, sg.inv);
        lim.y = sg.n_ctx + kvq_div(sg.r0 + c + 1, sg.rep, sg.inv);
        __syncthreads();
        r0.clear();
        r1.clear();
        top_all = 0;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
    }

    // One block at `kb` (K, then V), from position p0 on.
    template <bool MASKED>
    __device__ __forceinline__ void block(const uint8_t* kb, int p0) {
        const uint8_t* vb = kb + BLOCK;
        const int pos = p0 + g;
        auto seen = [&](int limit, int e) { return !MASKED || pos + 8 * e <= limit; };
        float2 x[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        {
            uint32_t w[W], s[NG];
            ka_words<W>(kb, lane, w);
            ka_scales<NG>(kb + CODES, g, s);
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                uint32_t a0[4], a1[4], q[4];
                if (BITS == 4) {
                    uint32_t u[4], v[4];
                    ka_nibbles(w[k], magic, u);
                    ka_nibbles(w[W / 2 + k], magic, v);
                    a0[0] = u[0]; a0[1] = v[0]; a0[2] = u[1]; a0[3] = v[1];
                    a1[0] = u[2]; a1[1] = v[2]; a1[2] = u[3]; a1[3] = v[3];
                } else {
                    ka_bytes(w[2 * k], magic, a0[0], a0[2]);
                    ka_bytes(w[W / 2 + 2 * k], magic, a0[1], a0[3]);
                    ka_bytes(w[2 * k + 1], magic, a1[0], a1[2]);
                    ka_bytes(w[W / 2 + 2 * k + 1], magic, a1[1], a1[3]);
                }
                const float s0 = ka_scale<NG>(s, 0, k), s1 = ka_scale<NG>(s, 1, k);
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                ka_lds4(q_at + k * 512, q);
                ka_mma(c, a0, q[0], q[1]);
                ka_mma(c, a1, q[2], q[3]);
                x[0].x = fmaf(c[0], s0, x[0].x);
                x[0].y = fmaf(c[1], s0, x[0].y);
                x[1].x = fmaf(c[2], s1, x[1].x);
                x[1].y = fmaf(c[3], s1, x[1].y);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // the high half's part and the low half's
            x[e].x += __shfl_xor_sync(0xFFFFFFFFu, x[e].x, 2);
            x[e].y += __shfl_xor_sync(0xFFFFFFFFu, x[e].y, 2);
        }
        uint32_t vs[NG];
        ka_scales<NG>(vb + CODES, g, vs);
        bool raise = ka_scale_above<HD>(vb + CODES, lane, top_all);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (!seen(lim.x, e)) x[e].x = -INFINITY;
            if (!seen(lim.y, e)) x[e].y = -INFINITY;
            raise |= x[e].x > r0.thr || x[e].y > r1.thr;
        }
        if (__any_sync(0xFFFFFFFFu, raise)) {
            float m0 = fmaxf(r0.m, fmaxf(x[0].x, x[1].x)), m1 = fmaxf(r1.m, fmaxf(x[0].y, x[1].y));
            uint32_t t0 = r0.top, t1 = r1.top;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t big = 0;
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    const int i = e * NG + k;
                    big = ka_scale_bits(i & 1 ? vs[i >> 1] >> 16 : vs[i >> 1], big);
                }
                if (seen(lim.x, e)) t0 = max(t0, big);
                if (seen(lim.y, e)) t1 = max(t1, big);
            }
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) {
                m0 = fmaxf(m0, __shfl_xor_sync(0xFFFFFFFFu, m0, s));
                m1 = fmaxf(m1, __shfl_xor_sync(0xFFFFFFFFu, m1, s));
                t0 = max(t0, __shfl_xor_sync(0xFFFFFFFFu, t0, s));
                t1 = max(t1, __shfl_xor_sync(0xFFFFFFFFu, t1, s));
            }
            const float f0 = r0.move(m0, t0, fr.x), f1 = r1.move(m1, t1, fr.y);
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                o[d][0] *= f0;
                o[d][1] *= f1;
                o[d][2] *= f0;
                o[d][3] *= f1;
            }
            top_all = __reduce_min_sync(0xFFFFFFFFu, min(r0.top, r1.top));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float2 y = ka_fma2(x[e], fr, make_float2(r0.nref, r1.nref));
            x[e] = make_float2(ka_exp2(y.x), ka_exp2(y.y));
            r0.l += x[e].x;
            r1.l += x[e].y;
        }
        uint32_t w[W];
        ka_words<W>(vb, lane, w);
        // columns from 4 on take what the high half leaves, times 2^11
        const float low = tq < 2 ? 0.f : -2048.f, up = tq < 2 ? 1.f : 2048.f;
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            uint32_t pf[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float sc = ka_scale<NG>(vs, e, k);
                float2 y = make_float2(x[e].x * sc, x[e].y * sc);
                if (MASKED) {  // an unseen position's scale may be NaN
                    if (!seen(lim.x, e)) y.x = 0.f;
                    if (!seen(lim.y, e)) y.y = 0.f;
                }
                const float2 z = ka_fma2(ka_unpack(ka_pack(y.x, y.y)), make_float2(low, low), ka_mul2(y, make_float2(up, up)));
                pf[e] = ka_trans(ka_pack(z.x, z.y));
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
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                ka_mma(c, v, pf[0], pf[1]);
                ka_add4(o[d], c);
            }
        }
    }

    // The warp's rows to slot [RT][HD], exponents and sums to stat; a warp that saw nothing says so by its exponent.
    __device__ __forceinline__ void store(float* slot, float* exps, float* sums) {
        const float out = tq < 2 ? 1.f : 0x1p-11f, out2 = BITS == 4 ? 0.0625f * out : out;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = 2 * tq + j;
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                float2 y = make_float2(o[d][j] * out, o[d][2 + j] * out2);
                y.x += __shfl_xor_sync(0xFFFFFFFFu, y.x, 2);
                y.y += __shfl_xor_sync(0xFFFFFFFFu, y.y, 2);
                if (row < RT) *reinterpret_cast<float2*>(slot + row * HD + 16 * d + 2 * g) = y;
            }
            KvqRow& r = j ? r1 : r0;
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) r.l += __shfl_xor_sync(0xFFFFFFFFu, r.l, s);
            if (g == 0 && row < RT) {
                exps[row] = r.none() ? -INFINITY : -r.nref;
                sums[row] = r.l;
            }
        }
    }
};

// Up to 8 rows (NR 1: row g of M is q's high half, row g + 8 its low half) or 16 (NR 2: rows g and g + 8, the halves one
// after the other).  A thread holds row g (and g + 8), positions 2 tq, 2 tq + 1 and 8 on of a block; of the output
// columns 2 tq and 2 tq + 1, dims 16 d + 2 g and one on.
template <int BITS, int HD, int NR>
struct ManyRows {
    static constexpr int RT = 8 * NR, NG = HD / 32, W = HD * BITS / 64, CODES = kvq_code_bytes(BITS, HD), BLOCK = kvq_block_bytes(BITS, HD);
    static constexpr int NQ = (NG + KA_WARPS - 1) / KA_WARPS;
    const uint8_t* q_at;
    int lane, g, tq;
    uint32_t magic;
    float fr[NR];
    int lim[NR];
    KvqRow r[NR];
    float o[NR][HD / 16][4];
    uint32_t top_all;

    // q to [NR][NG][2][lane] four registers
    __device__ __forceinline__ void load_q(const KvqAttnArgs& a, const KvqSeg& sg, uint8_t* qs, float* q_max, int warp, float log2e_d) {
        lane = threadIdx.x & 31;
        g = lane >> 2;
        tq = lane & 3;
        magic = ka_magic();
        q_at = qs + lane * 16;
        float x[NR][NQ][8];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const int row = nr * 8 + g;
            const bool valid = row < sg.rows;
            const float* qp = kvq_query(a, sg, valid ? row : 0, HD) + tq * 8;
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
            if (tq == 0) q_max[warp * RT + row] = mx;
        }
        __syncthreads();
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const int row = nr * 8 + g, sh = kvq_shift(kvq_row_max<RT>(q_max, row));
            const float sc = __int_as_float((sh + 127) << 23);
            fr[nr] = __int_as_float((127 - sh) << 23) * log2e_d;
            lim[nr] = sg.n_ctx + kvq_div(sg.r0 + row, sg.rep, sg.inv);
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                const int k = i * KA_WARPS + warp;
                if (k >= NG) continue;
                uint32_t hi[4], lo[4];
                kvq_split_q<BITS>(x[nr][i], sc, hi, lo);
                uint32_t* dst = reinterpret_cast<uint32_t*>(qs + k * 1024 + lane * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t* d = dst + (j >> 1) * 128 + (j & 1) * 2;
                    if (NR == 2) {
                        d[nr] = hi[j];
                        d[NG * 256 + nr] = lo[j];
                    } else {
                        d[0] = hi[j];
                        d[1] = lo[j];
                    }
                }
            }
            r[nr].clear();
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) o[nr][d][0] = o[nr][d][1] = o[nr][d][2] = o[nr][d][3] = 0.f;
        }
        top_all = 0;
        __syncthreads();
    }

    // The scales of positions 2 tq, 2 tq + 8, 2 tq + 1, 2 tq + 9, NG each, two to a word.
    __device__ __forceinline__ void scales(const uint8_t* p, uint32_t (&s)[2 * NG]) const {
#pragma unroll
        for (int i = 0; i < 2 * NG; i += NG % 2 ? 2 : 4) {
            if (NG % 2) ka_lds2(p + tq * (8 * NG) + 4 * i, &s[i]);
            else ka_lds4(p + tq * (8 * NG) + 4 * i, &s[i]);
        }
    }
    // Scale of group k of position 2 tq + e (e = 0, 1) or 2 tq + 6 + e (e = 2, 3).
    static __device__ __forceinline__ float scale(const uint32_t (&s)[2 * NG], int e, int k) {
        const int i = ((e & 1) * 2 + (e >> 1)) * NG + k;
        const __half2 h = *reinterpret_cast<const __half2*>(&s[i >> 1]);
        return i & 1 ? __high2float(h) : __low2float(h);
    }

    template <bool MASKED>
    __device__ __forceinline__ void block(const uint8_t* kb, int p0) {
        const uint8_t* vb = kb + BLOCK;
        auto seen = [&](int nr, int e) { return !MASKED || p0 + 2 * tq + (e & 1) + (e >> 1) * 8 <= lim[nr]; };
        float2 x[NR][2];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) x[nr][0] = x[nr][1] = make_float2(0.f, 0.f);
        {
            uint32_t w[W], s[2 * NG];
            ka_words<W>(kb, lane, w);
            scales(kb + CODES, s);
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                uint32_t qf[NR][2][4];
#pragma unroll
                for (int part = 0; part < NR; ++part) {
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
                    for (int part = NR - 1; part >= 0; --part) {  // the low halves first
                        ka_mma(c, qf[part][0], f[0], f[1]);
                        ka_mma(c, qf[part][1], f[2], f[3]);
                    }
                    const float2 sc = make_float2(scale(s, half * 2, k), scale(s, half * 2 + 1, k));
                    x[NR - 1][half] = ka_fma2(make_float2(c[2], c[3]), sc, x[NR - 1][half]);
                    x[0][half] = ka_fma2(make_float2(c[0], c[1]), sc, x[0][half]);
                }
            }
        }
        uint32_t vs[2 * NG];
        scales(vb + CODES, vs);
        bool raise = ka_scale_above<HD>(vb + CODES, lane, top_all);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (!seen(nr, 2 * e)) x[nr][e].x = -INFINITY;
                if (!seen(nr, 2 * e + 1)) x[nr][e].y = -INFINITY;
                raise |= x[nr][e].x > r[nr].thr || x[nr][e].y > r[nr].thr;
            }
        if (__any_sync(0xFFFFFFFFu, raise)) {
            uint32_t least = 0xFFFFu;
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                float mx = r[nr].m;
                uint32_t tp = r[nr].top;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    mx = fmaxf(mx, e & 1 ? x[nr][e >> 1].y : x[nr][e >> 1].x);
                    if (seen(nr, e)) {
#pragma unroll
                        for (int k = 0; k < NG; ++k) {
                            const int i = ((e & 1) * 2 + (e >> 1)) * NG + k;
                            tp = ka_scale_bits(i & 1 ? vs[i >> 1] >> 16 : vs[i >> 1], tp);
                        }
                    }
                }
#pragma unroll
                for (int s = 1; s < 4; s <<= 1) {
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, s));
                    tp = max(tp, __shfl_xor_sync(0xFFFFFFFFu, tp, s));
                }
                const float f = r[nr].move(mx, tp, fr[nr]);
                least = min(least, r[nr].top);
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
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float2 y = ka_fma2(x[nr][e], make_float2(fr[nr], fr[nr]), make_float2(r[nr].nref, r[nr].nref));
                x[nr][e] = make_float2(ka_exp2(y.x), ka_exp2(y.y));
                r[nr].l += x[nr][e].x + x[nr][e].y;
            }
        uint32_t w[W];
        ka_words<W>(vb, lane, w);
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            uint32_t hi[NR][2], lo[NR][2];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float2 y = ka_mul2(x[nr][e], make_float2(scale(vs, 2 * e, k), scale(vs, 2 * e + 1, k)));
                    if (MASKED) {  // an unseen position's scale may be NaN
                        if (!seen(nr, 2 * e)) y.x = 0.f;
                        if (!seen(nr, 2 * e + 1)) y.y = 0.f;
                    }
                    hi[nr][e] = ka_pack(y.x, y.y);
                    // what is left, times 2^11
                    const float2 z = ka_fma2(ka_unpack(hi[nr][e]), make_float2(-2048.f, -2048.f), ka_mul2(y, make_float2(2048.f, 2048.f)));
                    lo[nr][e] = ka_pack(z.x, z.y);
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
                for (int nr = 0; nr < NR; ++nr) {
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
                    ka_mma(c, v, lo[nr][0], lo[nr][1]);
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        const float2 low = ka_mul2(make_float2(c[i], c[i + 1]), make_float2(0x1p-11f, 0x1p-11f));
                        c[i] = low.x;
                        c[i + 1] = low.y;
                    }
                    ka_mma(c, v, hi[nr][0], hi[nr][1]);
                    ka_add4(o[nr][d], c);
                }
            }
        }
    }

    __device__ __forceinline__ void store(float* slot, float* exps, float* sums) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int d = 0; d < HD / 16; ++d)
                    *reinterpret_cast<float2*>(slot + (nr * 8 + 2 * tq + j) * HD + 16 * d + 2 * g) =
                        make_float2(o[nr][d][j], o[nr][d][2 + j] * (BITS == 4 ? 0.0625f : 1.0f));
            r[nr].l += __shfl_xor_sync(0xFFFFFFFFu, r[nr].l, 1);
            r[nr].l += __shfl_xor_sync(0xFFFFFFFFu, r[nr].l, 2);
            if (tq == 0) {
                exps[nr * 8 + g] = r[nr].none() ? -INFINITY : -r[nr].nref;
                sums[nr * 8 + g] = r[nr].l;
            }
        }
    }
};
template <int BITS, int HD, int MODE>
struct KvqCore {
    using type = ManyRows<BITS, HD, MODE>;
};
template <int BITS, int HD>
struct KvqCore<BITS, HD, 0> {
    using type = FewRows<BITS, HD>;
};

// CLUSTER: a cluster of pl.split CTAs per unit (all of them, from the sequences' T rows), which join over distributed
// shared memory; else ranges, and a second launch.
template <int BITS, int HD, int MODE, bool CLUSTER>
__global__ void __launch_bounds__(KA_THREADS, KvqCfg<BITS, HD, MODE>::CTAS)
tf_kvq_attn_kernel(const KvqAttnArgs a, const KvqPlan pl) {
    using F = KvqCfg<BITS, HD, MODE>;
    constexpr int RT = F::RT;
    extern __shared__ __align__(128) uint8_t smem[];
    if (!CLUSTER) pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring_at = warp * (F::ST * F::STAGE), ring = smem_u32(smem) + ring_at;
    uint8_t* qs = smem + KA_WARPS * F::RING;
    float* slot_all = reinterpret_cast<float*>(smem);  // where the rings are, once a segment's blocks are done
    float* stat = reinterpret_cast<float*>(qs + F::QS);  // [warp][RT] exponents, then sums, then q's maxima
    float* q_max = stat + 2 * KA_WARPS * RT;
    KvqDesc* desc = static_cast<KvqDesc*>(a.ws);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.ws) + KA_DESC_BYTES);

    KvqRange range = {0, 1, 0, 0, 0};
    int b = 0, base = 0, rank = 0;
    if (CLUSTER) {
        rank = blockIdx.x % pl.split;
        b = blockIdx.x / (pl.split * pl.tiles * a.n_kv);
    } else {
        range = kvq_range<RT>(a, pl);
        b = range.b;
        base = range.base;
    }
    KvqDesc open = {-1, 0, 0, 0, 0, 0};  // the unit that begins here and ends in a later CTA
    const float log2e_d = 1.4426950408889634f * rsqrtf((float)HD);
    typename KvqCore<BITS, HD, MODE>::type core;

#pragma unroll 1
    for (int gpos = range.g0; gpos < range.g1;) {
        KvqSeq sq = kvq_seq(a, pl.rep, RT, b);
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
                const int row = i / (HD / 4), rr = r0 + row, t = kvq_div(rr, pl.rep, pl.inv), h = kvh * pl.rep + rr - t * pl.rep;
                *reinterpret_cast<float4*>(a.out + ((long long)b * a.T + t) * a.ld_out + h * HD + (i - row * (HD / 4)) * 4) =
                    make_float4(0.f, 0.f, 0.f, 0.f);
            }
            rows = min(RT, sq.n_new * pl.rep - r0);
            if (rows <= 0) return;  // the whole cluster
        } else {
            int len = kvq_len(sq);
            while (gpos >= base + len && b + 1 < a.B) {  // gpos is below the total: a sequence with work follows
                base += len;
                sq = kvq_seq(a, pl.rep, RT, ++b);
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

        // this warp's blocks: blk0 + warp, and every KA_WARPS-th from there
        const int n_mine = blk1 - blk0 > warp ? (blk1 - blk0 - warp + KA_WARPS - 1) / KA_WARPS : 0;
        const long long where = sq.slot * a.slot_bytes + kvh * a.head_bytes + (long long)(blk0 + warp) * F::BLOCK + lane * 16;
        const uint8_t *kc = a.kc + where, *vc = a.vc + where;
        int left = n_mine;
        uint32_t fill = ring;
        auto fetch = [&]() {  // the next block into the next stage
            if (left > 0) {
                const uint32_t dst = fill + lane * 16;
#pragma unroll
                for (int c = 0; c < F::BLOCK; c += 512)
                    if (c + 512 <= F::BLOCK || lane * 16 < F::BLOCK - c) {
                        ka_copy16(dst + c, kc + c);
                        ka_copy16(dst + F::BLOCK + c, vc + c);
                    }
                --left;
                kc += KA_WARPS * F::BLOCK;
                vc += KA_WARPS * F::BLOCK;
                fill = fill == ring + (F::ST - 1) * F::STAGE ? ring : fill + F::STAGE;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < F::ST - 1; ++i) fetch();
        const KvqSeg sg = {b, kvh, r0, rows, pl.rep, a.T, sq.n_ctx, pl.inv, sq.n_ctx + kvq_div(r0, pl.rep, pl.inv)};
        core.load_q(a, sg, qs, q_max, warp, log2e_d);

        uint32_t at = ring_at;
        int p0 = (blk0 + warp) * 16;
#pragma unroll 1
        for (int i = 0; i < n_mine; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(F::ST - 2) : "memory");
            __syncwarp();  // everyone's copies of this stage are visible, and the stage before is read
            fetch();
            if (p0 + 15 <= sg.open_to) core.template block<false>(smem + at, p0);
            else core.template block<true>(smem + at, p0);
            p0 += KA_WARPS * 16;
            at = at == ring_at + (F::ST - 1) * F::STAGE ? ring_at : at + F::STAGE;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // the rings are read: the warps' rows take their place
        core.store(slot_all + warp * RT * HD, stat + warp * RT, stat + (KA_WARPS + warp) * RT);
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
                const int rr = r0 + row, t = kvq_div(rr, pl.rep, pl.inv), h = kvh * pl.rep + rr - t * pl.rep;
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
                const int rr = r0 + row, t = kvq_div(rr, pl.rep, pl.inv), h = kvh * pl.rep + rr - t * pl.rep;
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
        const KvqSeq sq = kvq_seq(a, pl.rep, RT, s);
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
    const KvqDesc de = static_cast<const KvqDesc*>(a.ws)[blockIdx.x];
    if (pl.by_unit) {  // a unit that does not exist has no descriptor
        const KvqSeq sq = kvq_seq(a, pl.rep, pl.rt, blockIdx.x / (a.n_kv * pl.tiles));
        if ((int)(blockIdx.x % pl.tiles) * a.n_kv >= sq.units) return;
    }
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
    const int rep = pl.rep, rr = de.tile * rt + r, t = kvq_div(rr, rep, pl.inv), h = de.kvh * rep + rr - t * rep;
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    *reinterpret_cast<float4*>(a.out + ((long long)de.b * a.T + t) * a.ld_out + h * hd + d) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// ---- host ------------------------------------------------------------------------------------------
static int kvq_sms() {
    static std::atomic<int> known[64] = {};  // per device: a quarter of a microsecond a call
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && known[dev].load() > 0) return known[dev].load();
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    sms = sms < 1 ? 1 : (4 * sms > KA_MAX_GRID ? KA_MAX_GRID / 4 : sms);
    if (dev >= 0 && dev < 64) known[dev].store(sms);
    return sms;
}

// CTAs per unit where a cluster takes each unit: as many as leave all units resident, while a warp has no more than
// KA_TURNS blocks at the cache's capacity (lengths are on the device; longer ones are balanced better by ranges).
// Clusters / ranges: 32 sequences of 5 new rows over 1144 positions (9 blocks a warp) 16.5 / 23.0 us, 4 of 8 over 2000 (8)
// 19.2 / 23.0, 1 of 4 over 8000 (16) 22.1 / 16.0, 3 of 1 over 9000 (18) 14.4 / 12.5.  Capacity stands for lengths that the host
// does not know: short contexts in a long cache take ranges (32 of 5 rows over 1144 in a cache of 8192: 22.9).  Clusters of 16
// gain 0 to 5 % from 3000 positions on and lose 20 % on the shortest calls.
constexpr int KA_TURNS = 10;
static int kvq_split_of(long long units, int cap, int slots) {
    if (units > slots) return 0;
    const int s = (int)(slots / units) < KA_MAX_SPLIT ? (int)(slots / units) : KA_MAX_SPLIT;
    return cap / 16 <= s * KA_WARPS * KA_TURNS ? s : 0;
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
    pl.inv = (unsigned)(((1ull << 32) + pl.rep - 1) / pl.rep);  // (1: not used)
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
    // few units have many parts each: eight warps to a row, else one, which has eight parts in flight
    if (units * 8 <= slots) return kvq_launch((const void*)tf_kvq_combine_kernel<1, 8>, dim3(found, F::RT), 256, 0, 1, args, st, true);
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
