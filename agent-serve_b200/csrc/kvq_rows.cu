// Rows of a quantised KV cache: per-head RMS norm of queries and keys with the rotation in the same pass,
// keys and values into Q4_0 / Q8_0 blocks, and rows read back.
//
//   norm    y = (x inv) w, inv = 1 / sqrt(mean x^2 + eps), the mean in 64 bits (the row norm's own order)
//   rotate  pairs (j, j + rot / 2): (a, b) -> (a c - b s, a s + b c), c and s the cosine and sine of
//           pos freq[j].  The angle is a product in 64 bits: in fp32 a far position's angle is off by
//           2^-24 of itself, 0.004 at 65536.  The two products are summed in 64 bits and rounded once, so that a
//           key next to the border of two codes takes the same code wherever it is computed.
//   Q4_0    scale = f16(m / -8), m the group's first value of largest magnitude; code = rint(x / scale) in [-8, 7]
//   Q8_0    scale = f16(max|x| r), r = 1 / 127 in fp32; code = rint(x / scale) in [-127, 127]
// (x / scale is IEEE's quotient: none rounds to a half that it is not, since a half times an f16 scale
// fits 19 bits.)  A group with an infinity or NaN gets a NaN for its scale and reads back as NaN; a
// scale beyond f16 is held at 65504, and a zero scale reads back as zeros.
//
// One warp per row and share of its heads; 8, 16 or 32 lanes per head, four dims each, so that a group of
// 32 is eight lanes.
#include "kvq.cuh"

namespace tfb {

constexpr int KR_THREADS = 256;
constexpr int KR_VEC = 4;  // vectors of a warp in flight

__device__ __forceinline__ int kvq_slot(const int* slots, int row) { return slots ? slots[row] : row; }

// Codes and scale of a group of 32 over eight neighbouring lanes, four values each.
template <int BITS>
__device__ __forceinline__ void quantise(const float4& x, int lane, int (&code)[4], __half& scale) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    const unsigned mine = top;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    float d;
    if (BITS == 4) {
        float m = v[3];
#pragma unroll
        for (int i = 2; i >= 0; --i)
            if ((__float_as_uint(v[i]) & 0x7FFFFFFFu) == top) m = v[i];
        const unsigned has = __ballot_sync(0xFFFFFFFFu, mine == top) >> (lane & 24) & 0xFFu;
        m = __shfl_sync(0xFFFFFFFFu, m, (lane & 24) + __ffs(has) - 1);
        d = __fmul_rn(m, -0.125f);
    } else {
        d = __fmul_rn(__uint_as_float(top), 1.0f / 127.0f);
    }
    const bool bad = top >= 0x7F800000u;
    scale = bad ? __ushort_as_half(0x7FFF) : __float2half_rn(fminf(fmaxf(d, -65504.0f), 65504.0f));
    const float s = __half2float(scale);
    const float lo = BITS == 4 ? -8.0f : -127.0f, hi = BITS == 4 ? 7.0f : 127.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        code[i] = (bad || s == 0.0f ? 0 : (int)fminf(fmaxf(rintf(__fdiv_rn(v[i], s)), lo), hi)) + (BITS == 4 ? 8 : 128);
}

// Four dims 4 hl .. 4 hl + 3 of position p of a block.
template <int BITS>
__device__ __forceinline__ void store_k(uint8_t* blk, int hd, int p, int hl, const int (&c)[4]) {
    const int half = p >> 3, lane = (p & 7) * 4 + (hl >> 1 & 3), words = hd * BITS / 64, grp = hl >> 3;
    if (BITS == 4)
        *reinterpret_cast<uint16_t*>(blk + kvq_word(words, half * (hd >> 5) + grp, lane) + (hl & 1) * 2) =
            (uint16_t)(c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12);
    else
        *reinterpret_cast<uint32_t*>(blk + kvq_word(words, half * (hd >> 4) + grp * 2 + (hl & 1), lane)) =
            (uint32_t)c[0] | (uint32_t)c[1] << 8 | (uint32_t)c[2] << 16 | (uint32_t)c[3] << 24;
}
template <int BITS>
__device__ __forceinline__ void store_v(uint8_t* blk, int hd, int p, int hl, const int (&c)[4]) {
    const int words = hd * BITS / 64, byte = (p & 1) * 2 + (p >> 3), tile = hl >> 2;
    const int lane = (hl & 3) * 8 + ((p & 7) >> 1);  // of dims 0 and 1; dims 2 and 3: four lanes on
    if (BITS == 4) {
        uint8_t* w = blk + kvq_word(words, tile, lane) + byte;
        const int next = tile < (words & ~3) ? 64 : 32;
        w[0] = (uint8_t)(c[0] | c[1] << 4);
        w[next] = (uint8_t)(c[2] | c[3] << 4);
    } else {
        uint8_t* w = blk + kvq_word(words, tile * 2, lane) + byte;
        w[0] = (uint8_t)c[0];
        w[4] = (uint8_t)c[1];
        w[64] = (uint8_t)c[2];
        w[68] = (uint8_t)c[3];
    }
}

// LH lanes per head.  A warp takes vectors (32 / LH heads) first, first + split, ... of its row's
// n_head + 2 n_kv heads.
template <int LH, int BITS>
__global__ void __launch_bounds__(KR_THREADS) tf_kvq_rows_kernel(const KvqRowsArgs a, int split) {
    constexpr int HPW = 32 / LH;
    const int lane = threadIdx.x & 31, hl = lane & (LH - 1);
    const long long task = ((long long)blockIdx.x * KR_THREADS + threadIdx.x) >> 5;
    const int row = (int)(task / split), first = (int)(task - (long long)row * split);
    if (row >= a.rows) return;
    const int pos = a.pos ? a.pos[row] : 0;
    uint8_t *kblk = nullptr, *vblk = nullptr;
    if (a.kc) {
        const int slot = kvq_slot(a.slots, row);
        if (slot < 0) return;
        if (slot >= a.n_slots || pos < 0 || pos >= a.cap) {
            if (first == 0 && lane == 0) atomicCAS(a.err, 0, slot >= a.n_slots ? ERR_BAD_TOKEN : ERR_POS);
            return;
        }
        const long long off = slot * a.slot_bytes + (long long)(pos >> 4) * kvq_block_bytes(BITS, a.hd);
        kblk = a.kc + off;
        vblk = a.vc + off;
    } else if (pos < 0) {
        return;
    }
    const int nq = a.q ? a.n_head : 0, nk = nq + (a.k ? a.n_kv : 0), nv = nk + (a.v ? a.n_kv : 0);
    const int d0 = hl * 4, half = a.rot >> 1;
    const bool live = d0 < a.hd, turn = a.freq && d0 < a.rot;
    // cosines and sines of the lane's four dims; the second half's sign
    double c[4], s[4];
    int mate = lane;
    if (turn) {
        const int j0 = d0 < half ? d0 : d0 - half;
        mate = d0 < half ? lane + (half >> 2) : lane - (half >> 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            double sn, cs;
            sincos((double)pos * (double)a.freq[j0 + i], &sn, &cs);
            c[i] = (double)(float)cs;
            s[i] = d0 < half ? -(double)(float)sn : (double)(float)sn;
        }
    }
    float4 wq = make_float4(1.f, 1.f, 1.f, 1.f), wk = wq;
    if (a.q_weight && live) wq = *reinterpret_cast<const float4*>(a.q_weight + d0);
    if (a.k_weight && live) wk = *reinterpret_cast<const float4*>(a.k_weight + d0);
    const double inv_n = 1.0 / a.hd;
    const int vectors = (nv + HPW - 1) / HPW, sub = lane / LH;
    for (int i0 = first; i0 < vectors; i0 += split * KR_VEC) {
        float4 x[KR_VEC];
#pragma unroll
        for (int u = 0; u < KR_VEC; ++u) {
            const int h = (i0 + u * split) * HPW + sub;
            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (h < nv && live) {
                const float* p = h < nq   ? a.q + (long long)row * a.ld_q + (long long)h * a.hd
                                 : h < nk ? a.k + (long long)row * a.ld_k + (long long)(h - nq) * a.hd
                                          : a.v + (long long)row * a.ld_v + (long long)(h - nk) * a.hd;
                x[u] = *reinterpret_cast<const float4*>(p + d0);
            }
        }
#pragma unroll
        for (int u = 0; u < KR_VEC; ++u) {
            if (i0 + u * split >= vectors) break;
            const int h = (i0 + u * split) * HPW + sub;
            const bool isq = h < nq, isk = !isq && h < nk, rotated = h < nk;
            float4 y = x[u];
            if (a.q_weight || a.k_weight) {
                double ss = fma((double)y.x, (double)y.x, fma((double)y.y, (double)y.y, fma((double)y.z, (double)y.z, (double)y.w * (double)y.w)));
#pragma unroll
                for (int o = LH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
                if ((isq && a.q_weight) || (isk && a.k_weight)) {
                    const float inv = __fdiv_rn(1.0f, __fsqrt_rn((float)(ss * inv_n) + a.eps));
                    const float4 w = isq ? wq : wk;
                    y.x = __fmul_rn(__fmul_rn(y.x, inv), w.x);
                    y.y = __fmul_rn(__fmul_rn(y.y, inv), w.y);
                    y.z = __fmul_rn(__fmul_rn(y.z, inv), w.z);
                    y.w = __fmul_rn(__fmul_rn(y.w, inv), w.w);
                }
            }
            if (a.freq) {
                float4 m;
                m.x = __shfl_sync(0xFFFFFFFFu, y.x, mate);
                m.y = __shfl_sync(0xFFFFFFFFu, y.y, mate);
                m.z = __shfl_sync(0xFFFFFFFFu, y.z, mate);
                m.w = __shfl_sync(0xFFFFFFFFu, y.w, mate);
                if (turn && rotated) {
                    y.x = (float)fma((double)y.x, c[0], (double)m.x * s[0]);
                    y.y = (float)fma((double)y.y, c[1], (double)m.y * s[1]);
                    y.z = (float)fma((double)y.z, c[2], (double)m.z * s[2]);
                    y.w = (float)fma((double)y.w, c[3], (double)m.w * s[3]);
                }
            }
            if (isq) {
                if (live) *reinterpret_cast<float4*>(a.q_out + (long long)row * a.ld_qo + (long long)h * a.hd + d0) = y;
            } else if (isk && a.k_out && live) {
                *reinterpret_cast<float4*>(a.k_out + (long long)row * a.ld_ko + (long long)(h - nq) * a.hd + d0) = y;
            }
            if (a.kc && __any_sync(0xFFFFFFFFu, !isq && h < nv)) {
                int code[4];
                __half scale;
                quantise<BITS>(y, lane, code, scale);
                if (!isq && h < nv && live) {
                    uint8_t* blk = (isk ? kblk : vblk) + (long long)(isk ? h - nq : h - nk) * a.head_bytes;
                    const int p = pos & 15;
                    if (isk) store_k<BITS>(blk, a.hd, p, hl, code);
                    else store_v<BITS>(blk, a.hd, p, hl, code);
                    if ((hl & 7) == 0)
                        reinterpret_cast<__half*>(blk + kvq_code_bytes(BITS, a.hd))[((p & 7) * 2 + (p >> 3)) * (a.hd >> 5) + (hl >> 3)] = scale;
                }
            }
        }
    }
}

// ---- reading back -------------------------------------------------------------------------------------
template <int LH, int BITS>
__global__ void __launch_bounds__(KR_THREADS) tf_kvq_read_kernel(const KvqReadArgs a, int split) {
    constexpr int HPW = 32 / LH;
    const int lane = threadIdx.x & 31, hl = lane & (LH - 1);
    const long long task = ((long long)blockIdx.x * KR_THREADS + threadIdx.x) >> 5;
    const int row = (int)(task / split), first = (int)(task - (long long)row * split);
    if (row >= a.rows) return;
    const int pos = a.pos[row], slot = kvq_slot(a.slots, row);
    if (slot < 0) return;
    if (slot >= a.n_slots || pos < 0 || pos >= a.cap) {
        if (first == 0 && lane == 0) atomicCAS(a.err, 0, slot >= a.n_slots ? ERR_BAD_TOKEN : ERR_POS);
        return;
    }
    const long long off = slot * a.slot_bytes + (long long)(pos >> 4) * kvq_block_bytes(BITS, a.hd);
    const int nk = a.k ? a.n_kv : 0, nv = nk + (a.v ? a.n_kv : 0);
    const int words = a.hd * BITS / 64, p = pos & 15, phalf = p >> 3, d0 = hl * 4;
    // where the lane's four codes lie in a block of K and of V
    const int kat = BITS == 4 ? kvq_word(words, phalf * (a.hd >> 5) + (hl >> 3), (p & 7) * 4 + (hl >> 1 & 3)) + (hl & 1) * 2
                              : kvq_word(words, phalf * (a.hd >> 4) + (hl >> 3) * 2 + (hl & 1), (p & 7) * 4 + (hl >> 1 & 3));
    const int vtile = hl >> 2, vlane = (hl & 3) * 8 + ((p & 7) >> 1);
    const int vat = kvq_word(words, BITS == 4 ? vtile : vtile * 2, vlane) + (p & 1) * 2 + phalf;
    const int vnext = BITS == 4 && vtile >= (words & ~3) ? 32 : 64;
    const int sat = kvq_code_bytes(BITS, a.hd) + 2 * (((p & 7) * 2 + phalf) * (a.hd >> 5) + (hl >> 3));
    if (d0 >= a.hd) return;
    for (int i0 = first; i0 * HPW < nv; i0 += split * KR_VEC) {
        uint32_t code[KR_VEC];
        float s[KR_VEC];
#pragma unroll
        for (int u = 0; u < KR_VEC; ++u) {
            const int h = (i0 + u * split) * HPW + lane / LH;
            if (h >= nv) continue;
            const bool isk = h < nk;
            const uint8_t* blk = (isk ? a.kc : a.vc) + off + (long long)(isk ? h : h - nk) * a.head_bytes;
            s[u] = __half2float(*reinterpret_cast<const __half*>(blk + sat));
            if (isk)
                code[u] = BITS == 4 ? *reinterpret_cast<const uint16_t*>(blk + kat) : *reinterpret_cast<const uint32_t*>(blk + kat);
            else if (BITS == 4)
                code[u] = blk[vat] | blk[vat + vnext] << 8;
            else
                code[u] = blk[vat] | blk[vat + 4] << 8 | blk[vat + 64] << 16 | (uint32_t)blk[vat + 68] << 24;
        }
#pragma unroll
        for (int u = 0; u < KR_VEC; ++u) {
            const int h = (i0 + u * split) * HPW + lane / LH;
            if (h >= nv) continue;
            const bool isk = h < nk;
            float4 y;
            constexpr int Z = BITS == 4 ? 8 : 128, M = BITS == 4 ? 15 : 255;
            y.x = (float)((int)(code[u] & M) - Z) * s[u];
            y.y = (float)((int)(code[u] >> BITS & M) - Z) * s[u];
            y.z = (float)((int)(code[u] >> 2 * BITS & M) - Z) * s[u];
            y.w = (float)((int)(code[u] >> 3 * BITS & M) - Z) * s[u];
            float* o = isk ? a.k + (long long)row * a.ld_k + (long long)h * a.hd : a.v + (long long)row * a.ld_v + (long long)(h - nk) * a.hd;
            *reinterpret_cast<float4*>(o + d0) = y;
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------
// Warps per row: one when rows alone fill the device (16 warps on each of its SMs), else a row's vectors are
// shared out so that few rows finish in one round of loads.
static int kvq_split(int rows, int vectors) {
    const int want = (148 * 16 + rows - 1) / rows;
    return want < 1 ? 1 : want > vectors ? vectors : want;
}

template <int LH, int BITS>
static cudaError_t rows_launch(const KvqRowsArgs& a, cudaStream_t st) {
    const int heads = (a.q ? a.n_head : 0) + (a.k ? a.n_kv : 0) + (a.v ? a.n_kv : 0);
    const int split = kvq_split(a.rows, (heads * LH + 31) / 32);
    const long long warps = (long long)a.rows * split, per = KR_THREADS / 32;
    tf_kvq_rows_kernel<LH, BITS><<<(unsigned)((warps + per - 1) / per), KR_THREADS, 0, st>>>(a, split);
    return cudaGetLastError();
}
template <int LH, int BITS>
static cudaError_t read_launch(const KvqReadArgs& a, cudaStream_t st) {
    const int heads = (a.k ? a.n_kv : 0) + (a.v ? a.n_kv : 0);
    const int split = kvq_split(a.rows, (heads * LH + 31) / 32);
    const long long warps = (long long)a.rows * split, per = KR_THREADS / 32;
    tf_kvq_read_kernel<LH, BITS><<<(unsigned)((warps + per - 1) / per), KR_THREADS, 0, st>>>(a, split);
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
