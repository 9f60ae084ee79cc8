// Rows of a quantised KV cache: per-head RMS norm of queries and keys with the rotation in the same pass,
// keys and values into Q4_0 / Q8_0 blocks, and rows read back.
//
//   norm    y = (x inv) w, inv = 1 / sqrt(mean x^2 + eps), the mean in 64 bits (the row norm's own order)
//   rotate  pairs (j, j + rot / 2): (a, b) -> (a c - b s, a s + b c), c and s the cosine and sine of
//           pos freq[j].  The angle is a product in 64 bits: in fp32 a far position's angle is off by
//           2^-24 of itself, 0.004 at 65536.  The two products and their sum are carried with their rounding
//           errors (Dekker's product by fma, Knuth's sum) and rounded once, in queries and in keys: pairs whose
//           products cancel keep their last bits, and a key next to the border of two codes takes the same code
//           wherever it is computed.  (A product and an fma, for queries alone: 9001 rows of 32 + 8 heads of 128 63.5
//           us instead of 69.1, and off by 2^-25 of the larger product.  In 64 bits it
//           would take 12 conversions a vector through a pipe of 4 lanes a cycle.)
//   Q4_0    scale = f16(m / -8), m the group's first value of largest magnitude; code = rint(x / scale) in [-8, 7]
//   Q8_0    scale = f16(max|x| r), r = 1 / 127 in fp32; code = rint(x / scale) in [-127, 127]
// A group with an infinity or NaN gets a NaN for its scale and reads back as NaN; a scale beyond f16 is held at
// 65504, and a zero scale reads back as zeros.
//
// One warp per row and share of its heads; 8, 16 or 32 lanes per head, four dims each, so that a group of
// 32 is eight lanes.  A word of V's codes holds four positions of a block (a "quad": 2 t, 2 t + 8, 2 t + 1,
// 2 t + 9), so values are taken four rows at a time: neighbouring rows of the call that lie in one block at
// rising positions (a run) share their quads out over the run's warps.  Row by row, the bytes of a head's V
// touch 16 lines an instruction.
//
// Bound by memory and by instructions.  Norm and rotation of 9001 rows of 32 + 8 heads of 128: 69.1 us, 5.3 TB/s (132
// instructions a vector, issue slots 64 %, DRAM 54 %).  The same with values and 8-bit writing, 5003 rows: 65.3 us (158 a
// vector, issue 55 %, 0.7 of a stall per issue for want of instructions: the kernel is long).  8192 rows of 8 heads of 64
// in 4 bits: 15.0 us to write (142 a vector, issue 70 %, ALU 57 %; a warp has only four, and spills 52 bytes a thread to have five
// CTAs an SM), 11.8 us to read, where a plain write of the same rows takes 6.5.  Reading 16384 rows of 8 heads of 128 in 8
// bits: 35.7 us, a plain write 20.9; the loads' latency (10 of 16 stalls per issue; a warp of values has one quad on its way).
#include <type_traits>

#include "kvq.cuh"

namespace tfb {

constexpr int KR_THREADS = 256;
constexpr int KR_VEC = 4;  // vectors of a warp in flight (a lane owns a group of one of four)

__device__ __forceinline__ float2 kr_mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 kr_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 kr_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
// y c + m s, rounded once (but for cases within 2^-46 of a tie)
__device__ __forceinline__ float2 kr_turn(float2 y, float2 c, float2 m, float2 s) {
    const float2 m1 = make_float2(-1.f, -1.f);
    const float2 p = kr_mul2(y, c), np = kr_mul2(p, m1), q = kr_mul2(m, s), nq = kr_mul2(q, m1);
    const float2 e = kr_add2(kr_fma2(y, c, np), kr_fma2(m, s, nq));  // what the products' roundings left out
    const float2 t = kr_add2(p, q), b = kr_add2(t, np), z = kr_fma2(b, m1, t);
    const float2 et = kr_add2(kr_fma2(z, m1, p), kr_fma2(b, m1, q));  // p + q = t + et
    return kr_add2(t, kr_add2(e, et));
}
__device__ __forceinline__ float kr_max_nan(float a, float b) {  // NaN if either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

__device__ __forceinline__ float kr_rcp(float x) {  // to 2^-23
    float d;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
    return d;
}

// Scales of the groups of 32, eight neighbouring lanes each, of four vectors.  The vectors are reduced together: at
// each of the first two steps a lane hands on the half of them that its partner keeps, so that a lane ends with one
// vector's group (vector `own_vector`) and works its scale out once, not four times.  inv is the scale's reciprocal; the
// result says that a group holds an infinity or NaN.
__device__ __forceinline__ int own_vector(int lane) { return lane >> 1 & 3; }
__device__ __forceinline__ int vector_owner(int lane, int u) { return (lane & 24) + 2 * u; }
template <class F>
__device__ __forceinline__ float reduce_groups(const float (&v)[4], int lane, F f) {
    const bool up = lane & 4, odd = lane & 2;
    const float k0 = f(up ? v[2] : v[0], __shfl_xor_sync(0xFFFFFFFFu, up ? v[0] : v[2], 4));
    const float k1 = f(up ? v[3] : v[1], __shfl_xor_sync(0xFFFFFFFFu, up ? v[1] : v[3], 4));
    const float k = f(odd ? k1 : k0, __shfl_xor_sync(0xFFFFFFFFu, odd ? k0 : k1, 2));
    return f(k, __shfl_xor_sync(0xFFFFFFFFu, k, 1));
}
template <int BITS>
__device__ __forceinline__ bool group_scales(const float4 (&x)[4], int lane, __half& scale, float& inv) {
    auto up = [](float a, float b) { return kr_max_nan(a, b); };
    auto down = [](float a, float b) { return fminf(a, b); };
    float top, d, v[4];
    if (BITS == 4) {
        // the larger of the group's largest and least; where they tie, whichever comes first
        float w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            v[u] = up(up(x[u].x, x[u].y), up(x[u].z, x[u].w));
            w[u] = down(down(x[u].x, x[u].y), down(x[u].z, x[u].w));
        }
        const float hi = reduce_groups(v, lane, up), lo = reduce_groups(w, lane, down);
        float m = hi >= -lo ? hi : lo;
        top = up(hi, -lo);
        const bool tie = hi == -lo && hi > 0.0f;
        if (__any_sync(0xFFFFFFFFu, tie)) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float a = __shfl_sync(0xFFFFFFFFu, hi, vector_owner(lane, u));
                float f = x[u].w;
                f = fabsf(x[u].z) == a ? x[u].z : f;
                f = fabsf(x[u].y) == a ? x[u].y : f;
                f = fabsf(x[u].x) == a ? x[u].x : f;
                const unsigned has = __ballot_sync(0xFFFFFFFFu, fabsf(f) == a) >> (lane & 24) & 0xFFu;
                f = __shfl_sync(0xFFFFFFFFu, f, (lane & 24) + (has ? __ffs(has) - 1 : 0));
                if (tie && own_vector(lane) == u) m = f;
            }
        }
        d = __fmul_rn(m, -0.125f);
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = up(up(fabsf(x[u].x), fabsf(x[u].y)), up(fabsf(x[u].z), fabsf(x[u].w)));
        top = reduce_groups(v, lane, up);
        d = __fmul_rn(top, 1.0f / 127.0f);
    }
    const bool bad = !(top < INFINITY);
    scale = bad ? __ushort_as_half(0x7FFF) : __float2half_rn(fminf(fmaxf(d, -65504.0f), 65504.0f));
    const float s = __half2float(scale);
    inv = s == 0.0f ? 0.0f : kr_rcp(s);
    return __any_sync(0xFFFFFFFFu, bad);
}
// Codes of vector u.  A code is the low 16 bits of code[i]; above them lies what packing drops.
//
// rint(x / scale) without a quotient: rint of the product with the reciprocal (off by 2.3e-5 at 127) is
// right unless the product is next to a half; there (one vector in 130 of random values) the remainder x - q scale,
// which is exact, says which integer is nearest.  Adding 1.5 2^23 rounds to an integer, ties to even, in the low bits.
template <int BITS>
__device__ __forceinline__ void vector_codes(const float4& x, int lane, int u, __half scale, float own_inv, bool bad, uint32_t (&code)[4]) {
    constexpr float LO = BITS == 4 ? -8.0f : -127.0f, HI = BITS == 4 ? 7.0f : 127.0f, Z = BITS == 4 ? 8.0f : 128.0f;
    constexpr float M = 12582912.0f + Z;
    const float v[4] = {x.x, x.y, x.z, x.w}, inv = __shfl_sync(0xFFFFFFFFu, own_inv, vector_owner(lane, u));
    bool doubt = bad;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float r = fminf(fmaxf(__fmul_rn(v[i], inv), LO), HI);
        const float t = __fadd_rn(r, M);
        doubt |= fabsf(__fadd_rn(r, -__fadd_rn(t, -M))) > 0.49997f;
        code[i] = __float_as_uint(t);
    }
    if (__any_sync(0xFFFFFFFFu, doubt)) {
        const float s = __half2float(__shfl_sync(0xFFFFFFFFu, scale, vector_owner(lane, u)));
        const bool none = !(fabsf(s) > 0.0f);  // zero, or NaN
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float r = fminf(fmaxf(__fmul_rn(v[i], inv), LO), HI);
            const float q = __fadd_rn(__fadd_rn(r, M), -M), e = __fmaf_rn(-q, s, v[i]), e2 = fabsf(e + e);
            const bool next = e2 > fabsf(s) || (e2 == fabsf(s) && ((int)q & 1));
            const float to = next ? (__float_as_int(e) ^ __float_as_int(s)) < 0 ? q - 1.0f : q + 1.0f : q;
            code[i] = __float_as_uint((none ? 0.0f : fminf(fmaxf(to, LO), HI)) + M);
        }
    }
}
// four codes of 8 bits to a word
__device__ __forceinline__ uint32_t kr_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Four dims 4 hl .. 4 hl + 3 of position p of a block.
template <int BITS>
__device__ __forceinline__ int k_place(int hd, int p, int hl) {
    const int half = p >> 3, lane = (p & 7) * 4 + (hl >> 1 & 3), words = hd * BITS / 64, grp = hl >> 3;
    return BITS == 4 ? kvq_word(words, half * (hd >> 5) + grp, lane) + (hl & 1) * 2
                     : kvq_word(words, half * (hd >> 4) + grp * 2 + (hl & 1), lane);
}
// The words of quad t that hold dims 4 hl and 4 hl + 1 (Q8_0: the second 4 bytes on); those of dims 4 hl + 2 and
// 4 hl + 3 lie *next bytes on.
template <int BITS>
__device__ __forceinline__ int v_place(int hd, int t, int hl, int* next) {
    const int words = hd * BITS / 64, tile = hl >> 2;
    *next = BITS == 8 || tile < (words & ~3) ? 64 : 32;
    return kvq_word(words, BITS == 4 ? tile : tile * 2, (hl & 3) * 8 + t);
}
__device__ __forceinline__ int scale_place(int bits, int hd, int p, int grp) {
    return kvq_code_bytes(bits, hd) + 2 * (((p & 7) * 2 + (p >> 3)) * (hd >> 5) + grp);
}

// Which rows share a block with a warp's own: the run's first row, its length, this row's index in it, and the
// block's positions that it holds (rows in rising order of position).
struct Run {
    int first, len, index;
    unsigned mask;
    __device__ __forceinline__ int row(int p) const {  // the row of position p of the block, or -1
        if (mask == 0xFFFFu) return first + p;
        return mask >> p & 1 ? first + __popc(mask & ((1u << p) - 1)) : -1;
    }
    __device__ __forceinline__ int quads() const {  // bit t: quad t holds a row
        const unsigned m = mask | mask >> 8;
        return (m & 3 ? 1 : 0) | (m & 12 ? 2 : 0) | (m & 48 ? 4 : 0) | (m & 192 ? 8 : 0);
    }
};
// The n-th quad of a set.
__device__ __forceinline__ int nth_quad(unsigned quads, int n) {
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < n) quads &= quads - 1;
    return __ffs(quads) - 1;
}
// i / n for n = 1 .. 4 and i below 2^13
__device__ __forceinline__ int small_div(int i, int n) { return i * (n == 4 ? 16384 : n == 3 ? 21846 : n == 2 ? 32768 : 65536) >> 16; }
// Position of byte i of a quad's words.
__device__ __forceinline__ int quad_pos(int t, int i) { return 2 * t + (i >> 1) + (i & 1) * 8; }

template <class A>
__device__ __forceinline__ int row_slot(const A& a, int row) { return a.slots ? a.slots[row] : row; }

// Slots and positions of the rows 15 back to 16 on, a lane each; the row's own are lane 15's.
struct Window {
    int slot, pos;
};
template <class A>
__device__ __forceinline__ Window load_window(const A& a, int row) {
    const int q = row - 15 + (int)(threadIdx.x & 31);
    Window w = {-1, -1};
    if (q >= 0 && q < a.rows) {
        w.slot = row_slot(a, q);
        w.pos = a.pos[q];
    }
    return w;
}
// The run of `row`, which lies in the cache.
__device__ __forceinline__ Run find_run(int row, int slot, int pos) {
    const int lane = threadIdx.x & 31;
    const int slot0 = __shfl_up_sync(0xFFFFFFFFu, slot, 1), pos0 = __shfl_up_sync(0xFFFFFFFFu, pos, 1);
    const bool on = lane > 0 && slot >= 0 && slot == slot0 && pos0 >= 0 && pos > pos0 && pos >> 4 == pos0 >> 4;
    const unsigned c = __ballot_sync(0xFFFFFFFFu, on);  // rows that go on with the run of the row before
    const int back = __clz(~(c << 16)), ahead = __ffs(~(c >> 16)) - 1;
    Run r;
    r.first = row - back;
    r.len = back + 1 + ahead;
    r.index = back;
    const bool in = lane >= 15 - back && lane <= 15 + ahead;
    r.mask = __reduce_or_sync(0xFFFFFFFFu, in ? 1u << (pos & 15) : 0u);
    return r;
}

// How a row is dealt out to warps.
struct RowSplit {
    int split, vsplit;         // warps for queries and keys, and for values
    int turn;                  // warp i's keys begin at vector i + turn, modulo split
    unsigned long long inv;    // 2^64 / (split + vsplit), rounded up (2 or more)
};
__device__ __forceinline__ unsigned task_row(unsigned task, const RowSplit& sp) {  // task / (split + vsplit)
    return sp.split + sp.vsplit == 1 ? task : (unsigned)__umul64hi(task, sp.inv);
}
static RowSplit row_split(int split, int vsplit, int q_vectors) {
    const unsigned n = (unsigned)(split + vsplit);
    return {split, vsplit, split ? (split - q_vectors % split) % split : 0, n > 1 ? ~0ull / n + 1 : 0};
}

// LH lanes per head.  A row has `split` warps for its queries and keys (vectors of 32 / LH heads: first, first +
// split, ...) and `vsplit` for its share of the run's values.
// KIND 0: rows are only written, 1: normed or copied, and written if there is a cache, 2: rotated too, without a cache, 3: with
// one.  (Kernels of their own are shorter and have fewer registers.  CTAs an SM, 9001 rows rotated 2 / 3 / 4: 73.8 / 69.1 / 82.3 us,
// 5003 stored and read 82.4 / 76.5 / 83.7, 8192 rows of 8 heads of 64 in 4 bits written and read 3 / 4 / 5: 28.1 / 26.1 / 25.6.)
template <int LH, int BITS, int KIND>
__global__ void __launch_bounds__(KR_THREADS, KIND >= 2 ? 3 : KIND == 1 ? 4 : 5) tf_kvq_rows_kernel(const KvqRowsArgs a, const RowSplit sp) {
    constexpr int HPW = 32 / LH;
    constexpr bool TURN = KIND >= 2, WRITE = KIND == 0, CACHE = KIND == 0 || KIND == 3;
    const int lane = threadIdx.x & 31, hl = lane & (LH - 1), sub = lane / LH;
    const unsigned task = blockIdx.x * (KR_THREADS / 32) + (threadIdx.x >> 5);
    const int row = (int)task_row(task, sp), split = sp.split, vsplit = sp.vsplit;
    const int first = (int)(task - (unsigned)row * (split + vsplit));
    if ((unsigned)row >= (unsigned)a.rows) return;
    Window win = {0, 0};
    int pos = 0, slot = 0;
    float4 ahead[KR_VEC];  // the first vectors of the warp's share, on their way while the position is
    if (first < split) {
        const float* in = !WRITE && a.q ? a.q + (long long)row * a.ld_q : a.k + (long long)row * a.ld_k;
        const int heads = !WRITE && a.q ? a.n_head : a.n_kv;
#pragma unroll
        for (int u = 0; u < KR_VEC; ++u) {
            const int h = (first + u * split) * HPW + sub;
            ahead[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (h < heads && hl * 4 < a.hd) ahead[u] = *reinterpret_cast<const float4*>(in + h * a.hd + hl * 4);
        }
        if (a.pos) pos = a.pos[row];
        if (CACHE || (KIND == 1 && a.kc)) slot = row_slot(a, row);
    } else {
        win = load_window(a, row);
        pos = __shfl_sync(0xFFFFFFFFu, win.pos, 15);
        slot = __shfl_sync(0xFFFFFFFFu, win.slot, 15);
    }
    long long off = 0;
    if (CACHE || (KIND == 1 && a.kc)) {
        if (slot < 0) return;
        if (slot >= a.n_slots || pos < 0 || pos >= a.cap) {
            if (first == 0 && lane == 0) atomicCAS(a.err, 0, slot >= a.n_slots ? ERR_BAD_TOKEN : ERR_POS);
            return;
        }
        off = slot * a.slot_bytes + (long long)(pos >> 4) * kvq_block_bytes(BITS, a.hd);
    } else if (pos < 0) {
        return;
    }
    const int d0 = hl * 4, half = a.rot >> 1;
    const bool live = d0 < a.hd;
    if (first < split) {
        // cosines and sines of the row's angles (a lane computes one or two), then of the lane's four dims
        const bool turn = TURN && d0 < a.rot;
        float4 c = make_float4(0.f, 0.f, 0.f, 0.f), s = c;
        int mate = lane;
        if (TURN) {
            float cs[2] = {0.f, 0.f}, sn[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (lane + 32 * i < half) {
                    double u, v;
                    sincos((double)pos * (double)a.freq[lane + 32 * i], &u, &v);
                    sn[i] = (float)u;
                    cs[i] = (float)v;
                }
            const bool upper = d0 >= half;  // the pair's second element
            const int j0 = turn ? (upper ? d0 - half : d0) : 0, from = j0 & 31;
            float t[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                t[i] = __shfl_sync(0xFFFFFFFFu, cs[0], from + i);
                t[4 + i] = __shfl_sync(0xFFFFFFFFu, sn[0], from + i);
                if (half > 32) {
                    const float c1 = __shfl_sync(0xFFFFFFFFu, cs[1], from + i), s1 = __shfl_sync(0xFFFFFFFFu, sn[1], from + i);
                    if (j0 >= 32) {
                        t[i] = c1;
                        t[4 + i] = s1;
                    }
                }
                if (!upper) t[4 + i] = -t[4 + i];
            }
            c = make_float4(t[0], t[1], t[2], t[3]);
            s = make_float4(t[4], t[5], t[6], t[7]);
            if (turn) mate = upper ? lane - (half >> 2) : lane + (half >> 2);
        }
        const double inv_n = 1.0 / a.hd;
        // Vectors of one kind: the warp's, of `heads` heads from `in` on (its dims), to `out` and to the cache (`blk`)
        auto vectors_of = [&](auto is_k, const float* in, float* out, int heads, const float* weight, uint8_t* blk, int begin, bool loaded) {
            constexpr bool IS_K = decltype(is_k)::value;
            float4 w = make_float4(1.f, 1.f, 1.f, 1.f);
            const bool norm = !WRITE && weight;
            if (norm && live) w = *reinterpret_cast<const float4*>(weight + d0);
            const int step = split * HPW;
            int h = begin * HPW + sub;
            const int kat = k_place<BITS>(a.hd, pos & 15, hl), sat = scale_place(BITS, a.hd, pos & 15, hl >> 3);
            auto load = [&](int h0) {
#pragma unroll
                for (int u = 0; u < KR_VEC; ++u) {
                    ahead[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (h0 + u * step < heads && live) ahead[u] = *reinterpret_cast<const float4*>(in + (h0 + u * step) * a.hd);
                }
            };
            if (!loaded) load(h);
            for (int left = (heads + HPW - 1) / HPW - begin; left > 0; left -= split * KR_VEC, h += step * KR_VEC) {
                float4 x[KR_VEC];
#pragma unroll
                for (int u = 0; u < KR_VEC; ++u) x[u] = ahead[u];
                if (TURN || left > split * KR_VEC) load(h + step * KR_VEC);
                // The squares of the four vectors are summed together: at each of the first two steps a lane hands on
                // the half of its sums that its partner keeps, so that a lane ends with the sum of one of them.
                float inv = 1.0f;
                if (norm) {
                    double ss[KR_VEC];
#pragma unroll
                    for (int u = 0; u < KR_VEC; ++u) {
                        const float4 y = x[u];
                        ss[u] = fma((double)y.x, (double)y.x,
                                    fma((double)y.y, (double)y.y, fma((double)y.z, (double)y.z, (double)y.w * (double)y.w)));
                    }
                    const bool hi = lane & LH / 2, odd = lane & LH / 4;
                    const double e0 = hi ? ss[0] : ss[2], e1 = hi ? ss[1] : ss[3];
                    const double k0 = (hi ? ss[2] : ss[0]) + __shfl_xor_sync(0xFFFFFFFFu, e0, LH / 2);
                    const double k1 = (hi ? ss[3] : ss[1]) + __shfl_xor_sync(0xFFFFFFFFu, e1, LH / 2);
                    double sum = (odd ? k1 : k0) + __shfl_xor_sync(0xFFFFFFFFu, odd ? k0 : k1, LH / 4);
#pragma unroll
                    for (int o = LH / 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
                    inv = __fdiv_rn(1.0f, __fsqrt_rn((float)(sum * inv_n) + a.eps));
                }
#pragma unroll
                for (int u = 0; u < KR_VEC; ++u) {
                    if (left - u * split <= 0) continue;
                    const bool mine = h + u * step < heads && live;
                    float4& y = x[u];
                    if (norm) {
                        const float f = __shfl_sync(0xFFFFFFFFu, inv, (lane & ~(LH / 2 + LH / 4)) + (u >> 1) * (LH / 2) + (u & 1) * (LH / 4));
                        y.x = __fmul_rn(__fmul_rn(y.x, f), w.x);
                        y.y = __fmul_rn(__fmul_rn(y.y, f), w.y);
                        y.z = __fmul_rn(__fmul_rn(y.z, f), w.z);
                        y.w = __fmul_rn(__fmul_rn(y.w, f), w.w);
                    }
                    if (TURN) {
                        float4 m;
                        m.x = __shfl_sync(0xFFFFFFFFu, y.x, mate);
                        m.y = __shfl_sync(0xFFFFFFFFu, y.y, mate);
                        m.z = __shfl_sync(0xFFFFFFFFu, y.z, mate);
                        m.w = __shfl_sync(0xFFFFFFFFu, y.w, mate);
                        if (turn) {
                            const float2 r0 = kr_turn(make_float2(y.x, y.y), make_float2(c.x, c.y), make_float2(m.x, m.y), make_float2(s.x, s.y));
                            const float2 r1 = kr_turn(make_float2(y.z, y.w), make_float2(c.z, c.w), make_float2(m.z, m.w), make_float2(s.z, s.w));
                            float4 z = make_float4(r0.x, r0.y, r1.x, r1.y);
                            if (!(kr_max_nan(kr_max_nan(fabsf(z.x), fabsf(z.y)), kr_max_nan(fabsf(z.z), fabsf(z.w))) < INFINITY)) {
                                // an infinity's rounding error is NaN
                                if (!(fabsf(z.x) < INFINITY)) z.x = __fmaf_rn(y.x, c.x, __fmul_rn(m.x, s.x));
                                if (!(fabsf(z.y) < INFINITY)) z.y = __fmaf_rn(y.y, c.y, __fmul_rn(m.y, s.y));
                                if (!(fabsf(z.z) < INFINITY)) z.z = __fmaf_rn(y.z, c.z, __fmul_rn(m.z, s.z));
                                if (!(fabsf(z.w) < INFINITY)) z.w = __fmaf_rn(y.w, c.w, __fmul_rn(m.w, s.w));
                            }
                            y = z;
                        }
                    }
                    if (!WRITE && out && mine) *reinterpret_cast<float4*>(out + (h + u * step) * a.hd) = y;
                }
                if (WRITE || (IS_K && (CACHE || (KIND == 1 && blk)))) {
                    __half scale;
                    float back;
                    const bool bad = group_scales<BITS>(x, lane, scale, back);
                    const int own = h + own_vector(lane) * step;
                    if (own < heads && live && (hl & 1) == 0) *reinterpret_cast<__half*>(blk + own * a.head_bytes + sat) = scale;
#pragma unroll
                    for (int u = 0; u < KR_VEC; ++u) {
                        if (left - u * split <= 0) continue;
                        uint32_t code[4];
                        vector_codes<BITS>(x[u], lane, u, scale, back, bad, code);
                        if (h + u * step < heads && live) {
                            uint8_t* to = blk + (h + u * step) * a.head_bytes;
                            if (BITS == 4) *reinterpret_cast<uint16_t*>(to + kat) = (uint16_t)(code[0] + 16 * code[1] + 256 * code[2] + 4096 * code[3]);
                            else *reinterpret_cast<uint32_t*>(to + kat) = kr_bytes(code[0], code[1], code[2], code[3]);
                        }
                    }
                }
            }
        };
        if (!WRITE && a.q)
            vectors_of(std::false_type(), a.q + (long long)row * a.ld_q + d0, a.q_out + (long long)row * a.ld_qo + d0, a.n_head, a.q_weight,
                       nullptr, first, true);
        // keys go on where the queries' share ended, so that a row's warps have equal shares
        if (WRITE || a.k) {
            const int begin = first + sp.turn - (first + sp.turn >= split ? split : 0);
            vectors_of(std::true_type(), a.k + (long long)row * a.ld_k + d0, a.k_out ? a.k_out + (long long)row * a.ld_ko + d0 : nullptr, a.n_kv,
                       a.k_weight, a.kc ? a.kc + off : nullptr, begin, WRITE || !a.q);
        }
        return;
    }

    if (KIND == 2) return;  // (no values)
    // values: (quad, vector) pairs of the run, dealt out to its warps
    const Run run = find_run(row, win.slot, win.pos);
    const int quads = run.quads(), nquad = __popc(quads), vv = (a.n_kv + HPW - 1) / HPW;
    for (int i = run.index * vsplit + first - split; i < nquad * vv; i += run.len * vsplit) {
        const int vec = small_div(i, nquad), t = nth_quad(quads, i - vec * nquad), h = vec * HPW + sub;
        float4 x[4];
        bool all = true;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = run.row(quad_pos(t, j));
            x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            all = all && r >= 0;
            if (r >= 0 && h < a.n_kv && live) x[j] = *reinterpret_cast<const float4*>(a.v + (long long)r * a.ld_v + h * a.hd + d0);
        }
        uint8_t* blk = a.vc + off + h * a.head_bytes;
        __half scale;
        float back;
        const bool bad = group_scales<BITS>(x, lane, scale, back);
        const int own = quad_pos(t, own_vector(lane));
        if ((run.mask >> own & 1) && h < a.n_kv && live && (hl & 1) == 0)
            *reinterpret_cast<__half*>(blk + scale_place(BITS, a.hd, own, hl >> 3)) = scale;
        uint32_t w[4] = {0, 0, 0, 0};  // bytes of dims 0 and 1, and 2 and 3 (Q8_0: a word each)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t code[4];
            vector_codes<BITS>(x[j], lane, j, scale, back, bad, code);
#pragma unroll
            for (int e = 0; e < (BITS == 4 ? 2 : 4); ++e)  // byte j of word e
                w[e] = __byte_perm(w[e], BITS == 4 ? code[2 * e & 3] + 16 * code[(2 * e + 1) & 3] : code[e & 3], j == 0 ? 0x3214 : j == 1 ? 0x3240 : j == 2 ? 0x3410 : 0x4210);
        }
        if (h >= a.n_kv || !live) continue;
        int next;
        uint8_t* at = blk + v_place<BITS>(a.hd, t, hl, &next);
        if (all) {
            if (BITS == 4) {
                *reinterpret_cast<uint32_t*>(at) = w[0];
                *reinterpret_cast<uint32_t*>(at + next) = w[1];
            } else {
                *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
                *reinterpret_cast<uint2*>(at + next) = make_uint2(w[2], w[3]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!(run.mask >> quad_pos(t, j) & 1)) continue;
                if (BITS == 4) {
                    at[j] = (uint8_t)(w[0] >> 8 * j);
                    at[next + j] = (uint8_t)(w[1] >> 8 * j);
                } else {
                    at[j] = (uint8_t)(w[0] >> 8 * j);
                    at[4 + j] = (uint8_t)(w[1] >> 8 * j);
                    at[next + j] = (uint8_t)(w[2] >> 8 * j);
                    at[next + 4 + j] = (uint8_t)(w[3] >> 8 * j);
                }
            }
        }
    }
}

// ---- reading back -------------------------------------------------------------------------------------
// Values of four codes; a code as the low bits of 2^23 + code is exact, without a conversion.
template <int BITS>
__device__ __forceinline__ float4 kr_values(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, float s) {
    constexpr float Z = 8388608.0f + (BITS == 4 ? 8.0f : 128.0f);
    return make_float4((__uint_as_float(c0) - Z) * s, (__uint_as_float(c1) - Z) * s, (__uint_as_float(c2) - Z) * s, (__uint_as_float(c3) - Z) * s);
}
// 2^23 + byte j of x, or its low or high half
__device__ __forceinline__ uint32_t kr_byte(uint32_t x, int j) { return __byte_perm(x, 0x4B000000u, 0x7650 + j); }
__device__ __forceinline__ uint32_t kr_nibble(uint32_t x, int j) { return (x >> 4 * j & 15u) | 0x4B000000u; }

template <int LH, int BITS>
__global__ void __launch_bounds__(KR_THREADS) tf_kvq_read_kernel(const KvqReadArgs a, const RowSplit sp) {
    constexpr int HPW = 32 / LH;
    const int lane = threadIdx.x & 31, hl = lane & (LH - 1), sub = lane / LH;
    const unsigned task = blockIdx.x * (KR_THREADS / 32) + (threadIdx.x >> 5);
    const int row = (int)task_row(task, sp), split = sp.split, vsplit = sp.vsplit;
    const int first = (int)(task - (unsigned)row * (split + vsplit));
    if ((unsigned)row >= (unsigned)a.rows) return;
    Window win = {0, 0};
    int pos, slot;
    if (first < split) {
        pos = a.pos[row];
        slot = row_slot(a, row);
    } else {
        win = load_window(a, row);
        pos = __shfl_sync(0xFFFFFFFFu, win.pos, 15);
        slot = __shfl_sync(0xFFFFFFFFu, win.slot, 15);
    }
    if (slot < 0) return;
    if (slot >= a.n_slots || pos < 0 || pos >= a.cap) {
        if (first == 0 && lane == 0) atomicCAS(a.err, 0, slot >= a.n_slots ? ERR_BAD_TOKEN : ERR_POS);
        return;
    }
    const long long off = slot * a.slot_bytes + (long long)(pos >> 4) * kvq_block_bytes(BITS, a.hd);
    const int d0 = hl * 4, vectors = (a.n_kv + HPW - 1) / HPW;
    const bool live = d0 < a.hd;
    if (first < split) {
        const int kat = k_place<BITS>(a.hd, pos & 15, hl), sat = scale_place(BITS, a.hd, pos & 15, hl >> 3);
        for (int i0 = first; i0 < vectors; i0 += split * KR_VEC) {
            uint32_t code[KR_VEC];
            float s[KR_VEC];
#pragma unroll
            for (int u = 0; u < KR_VEC; ++u) {
                const int h = (i0 + u * split) * HPW + sub;
                if (h >= a.n_kv || !live) continue;
                const uint8_t* blk = a.kc + off + h * a.head_bytes;
                s[u] = __half2float(*reinterpret_cast<const __half*>(blk + sat));
                code[u] = BITS == 4 ? *reinterpret_cast<const uint16_t*>(blk + kat) : *reinterpret_cast<const uint32_t*>(blk + kat);
            }
#pragma unroll
            for (int u = 0; u < KR_VEC; ++u) {
                const int h = (i0 + u * split) * HPW + sub;
                if (h >= a.n_kv || !live) continue;
                const uint32_t c = code[u];
                *reinterpret_cast<float4*>(a.k + (long long)row * a.ld_k + h * a.hd + d0) =
                    BITS == 4 ? kr_values<4>(kr_nibble(c, 0), kr_nibble(c, 1), kr_nibble(c, 2), kr_nibble(c, 3), s[u])
                              : kr_values<8>(kr_byte(c, 0), kr_byte(c, 1), kr_byte(c, 2), kr_byte(c, 3), s[u]);
            }
        }
        return;
    }
    const Run run = find_run(row, win.slot, win.pos);
    const int quads = run.quads(), nquad = __popc(quads);
    for (int i = run.index * vsplit + first - split; i < nquad * vectors; i += run.len * vsplit) {
        const int vec = small_div(i, nquad), t = nth_quad(quads, i - vec * nquad), h = vec * HPW + sub;
        if (h >= a.n_kv || !live) continue;
        const uint8_t* blk = a.vc + off + h * a.head_bytes;
        int next;
        const uint8_t* at = blk + v_place<BITS>(a.hd, t, hl, &next);
        uint32_t w[4];
        if (BITS == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(at);
            w[1] = *reinterpret_cast<const uint32_t*>(at + next);
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(at), v = *reinterpret_cast<const uint2*>(at + next);
            w[0] = u.x; w[1] = u.y; w[2] = v.x; w[3] = v.y;
        }
        float s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = __half2float(*reinterpret_cast<const __half*>(blk + scale_place(BITS, a.hd, quad_pos(t, j), hl >> 3)));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = run.row(quad_pos(t, j));
            if (r < 0) continue;
            *reinterpret_cast<float4*>(a.v + (long long)r * a.ld_v + h * a.hd + d0) =
                BITS == 4 ? kr_values<4>(kr_nibble(w[0], 2 * j), kr_nibble(w[0], 2 * j + 1), kr_nibble(w[1], 2 * j), kr_nibble(w[1], 2 * j + 1), s[j])
                          : kr_values<8>(kr_byte(w[0], j), kr_byte(w[1], j), kr_byte(w[2], j), kr_byte(w[3], j), s[j]);
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------
// Warps per row: one when rows alone fill the device (`fill` warps on each of its SMs), else a row's vectors are
// shared out so that few rows finish in one round of loads.  16 warps, and twice what an SM holds where they carry
// a whole row of queries and keys, whose last round would else be long: 5003 rows of 32 + 8 + 8 heads of 128 written
// in 8 bits and read back, 79.5 us with 16, 76.5 with 48.
constexpr int KR_FILL = 16, KR_FILL_TURN = 48;
static int kvq_split(int rows, int vectors, int fill = KR_FILL) {
    const int want = (int)((148ll * fill + rows - 1) / rows);
    return want < 1 ? 1 : want > vectors ? vectors : want;
}

template <int LH, int BITS>
static cudaError_t rows_launch(const KvqRowsArgs& a, cudaStream_t st) {
    const int hpw = 32 / LH, q_vectors = a.q ? (a.n_head + hpw - 1) / hpw : 0, vectors = q_vectors + (a.k ? (a.n_kv + hpw - 1) / hpw : 0);
    const int split = vectors ? kvq_split(a.rows, vectors, a.freq ? KR_FILL_TURN : KR_FILL) : 0, vsplit = a.v ? kvq_split(a.rows, (a.n_kv * LH + 31) / 32) : 0;
    const RowSplit sp = row_split(split, vsplit, q_vectors);
    const long long warps = (long long)a.rows * (split + vsplit), per = KR_THREADS / 32;  // below 2^32: kvq_split
    const unsigned grid = (unsigned)((warps + per - 1) / per);
    const bool write = !a.q && !a.k_out && !a.k_weight;
    if (a.freq && a.kc) tf_kvq_rows_kernel<LH, BITS, 3><<<grid, KR_THREADS, 0, st>>>(a, sp);
    else if (a.freq) tf_kvq_rows_kernel<LH, 4, 2><<<grid, KR_THREADS, 0, st>>>(a, sp);
    else if (!write) tf_kvq_rows_kernel<LH, BITS, 1><<<grid, KR_THREADS, 0, st>>>(a, sp);
    else tf_kvq_rows_kernel<LH, BITS, 0><<<grid, KR_THREADS, 0, st>>>(a, sp);
    return cudaGetLastError();
}
template <int LH, int BITS>
static cudaError_t read_launch(const KvqReadArgs& a, cudaStream_t st) {
    const int each = kvq_split(a.rows, (a.n_kv * LH + 31) / 32), split = a.k ? each : 0, vsplit = a.v ? each : 0;
    const long long warps = (long long)a.rows * (split + vsplit), per = KR_THREADS / 32;
    tf_kvq_read_kernel<LH, BITS><<<(unsigned)((warps + per - 1) / per), KR_THREADS, 0, st>>>(a, row_split(split, vsplit, 0));
    return cudaGetLastError();
}

cudaError_t kvq_rows_launch(const KvqRowsArgs& a, cudaStream_t st) {
    if (a.hd <= 32) return a.bits == 4 ? rows_launch<8, 4>(a, st) : rows_launch<8, 8>(a, st);
    if (a.hd <= 64) return a.bits == 4 ? rows_launch<16, 4>(a, st) : rows_launch<16, 8>(a, st);
    return a.bits == 4 ? rows_launch<32, 4>(a, st) : rows_launch<32, 8>(a, st);
}
cudaError_t kvq_read_launch(const KvqReadArgs& a, cudaStream_t st) {
    if (a.hd <= 32) return a.bits == 4 ? read_launch<8, 4>(a, st) : read_launch<8, 8>(a, st);
    if (a.hd <= 64) return a.bits == 4 ? read_launch<16, 4>(a, st) : read_launch<16, 8>(a, st);
    return a.bits == 4 ? read_launch<32, 4>(a, st) : read_launch<32, 8>(a, st);
}

}  // namespace tfb
