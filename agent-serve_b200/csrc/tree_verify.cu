// Verification of a tree of drafted tokens against the target's distribution.
//
// p = softmax(logits / temperature) of a node's row, q = softmax(draft / temperature).  The walk
// starts at the root and tries the node's children in index order.  With a draft distribution
// (the children are draws from q), child x is accepted when u W q(x) < max(p(x) - c q(x), 0),
// c = 0 and W = 1 at first.  A rejection leaves the residual max(p' - q, 0), normalised, where
// p' = max(p - c q, 0) / W is the distribution so far; since
//     max(max(p - c q, 0) / W - q, 0) = max(p - (c + W) q, 0) / W,
// that is the same form with c' = c + W and W' = sum max(p - c' q, 0).  A residual without mass
// (p and q equal up to rounding) falls back to p.  Without a draft distribution child x is
// accepted when u W < p(x), and a rejection takes x out of p (W' = W - p(x)).  Temperature 0
// accepts the argmax (the first of equal ones).  When no child is accepted the next token is the
// first i whose cumulative residual exceeds u[root] times the residual's total.
//
// A pick by a cumulative sum over 10^5 terms is a discontinuous function of the terms: the
// exponentials are 32-bit, relative to the row's true maximum, every sum and residual is held in
// 64 bits.
//
// One thread-block cluster per sequence reads only the rows that its walk visits; each CTA has a
// contiguous slice of the vocabulary, each warp a contiguous piece of the slice.  A visited row
// takes two passes (maximum, sums; the second one from L2) with one exchange of C values through
// distributed shared memory after each; a rejection with a draft distribution and the final pick
// take one more pass each.  Every CTA holds the same sums in the same order and so takes the same
// decisions.
#include <cooperative_groups.h>

#include <atomic>

#include "tree.cuh"

namespace cg = cooperative_groups;

namespace tfb {

constexpr int TV_THREADS = 512;
constexpr int TV_WARPS = TV_THREADS / 32;
constexpr int TV_MAX_CLUSTER = 16;

// exp(l / temp - max): 1 at the maximum itself (also an infinite one); a NaN logit weighs nothing
__device__ __forceinline__ float tv_weight(float l, float mx, float inv_temp) {
    const float e = expf(__fmul_rn(__fsub_rn(l, mx), inv_temp));
    return l == mx ? 1.f : (l != l ? 0.f : e);
}

struct TvShared {
    double ex[2][TV_MAX_CLUSTER][2];   // exchanged values of the cluster's CTAs, two exchanges
    double red[TV_WARPS][2];
    unsigned long long key[TV_WARPS];
    int par[TREE_MAX_NODES], tok[TREE_MAX_NODES];
    float u[TREE_MAX_NODES];
    float2 child[TREE_MAX_NODES];      // logits of the current node's children: target, draft
    unsigned kids[TREE_MAX_NODES / 32];
    int gone[TREE_MAX_NODES];          // tokens taken out of p at this node
    int pick;
};

// N elements of a row from element i on, aligned when VEC (N = 4)
template <int N>
__device__ __forceinline__ void tv_load(float (&x)[N], const float* p) {
    if (N == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        x[0] = v.x, x[1 % N] = v.y, x[2 % N] = v.z, x[3 % N] = v.w;
    } else {
        x[0] = *p;
    }
}

template <int N, bool DRAFT>
__global__ void __launch_bounds__(TV_THREADS, 2) tf_tree_verify_kernel(const __grid_constant__ TreeVerifyArgs a, int slice, int piece) {
    extern __shared__ uint32_t out_bits[];  // without a draft distribution: the slice's tokens that are out of p
    __shared__ TvShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int b = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = a.V;
    const int n = a.n_node ? min(max(a.n_node[b], 0), a.T) : a.T;
    int* path = a.path + (size_t)b * a.T;
    if (n == 0) {
        if (rank == 0) {
            for (int i = tid; i < a.T; i += TV_THREADS) path[i] = -1;
            if (tid == 0) {
                a.n_path[b] = 0;
                a.next[b] = -1;
            }
        }
        return;
    }
    const bool greedy = a.inv_temp == 0.f;
    if (tid < n) {
        sh.par[tid] = a.parents[(size_t)b * a.T + tid];
        sh.tok[tid] = a.tokens[(size_t)b * a.T + tid];
        sh.u[tid] = greedy ? 0.f : a.u[(size_t)b * a.T + tid];
    }
    if (!DRAFT)
        for (int i = tid; i < (slice + 31) / 32; i += TV_THREADS) out_bits[i] = 0;
    __syncthreads();

    // this warp's elements: [w0, w1) of the row
    const int s0 = min(V, rank * slice), s1 = min(V, s0 + slice);
    const int w0 = min(s1, s0 + warp * piece), w1 = min(s1, w0 + piece);
    int parity = 0;
    // the cluster's values of `mine` (two per CTA), by rank, after one barrier
    auto exchange = [&](double x, double y) {
        parity ^= 1;
        if (tid < C) {
            double* o = cluster.map_shared_rank(&sh.ex[parity][rank][0], tid);
            o[0] = x;
            o[1] = y;
        }
        cluster.sync();
    };
    // block sums of two doubles (every thread gets them)
    auto block_sum = [&](double& x, double& y) {
        x = warp_sum_d(x);
        if (DRAFT) y = warp_sum_d(y);
        __syncthreads();
        if (lane == 0) {
            sh.red[warp][0] = x;
            sh.red[warp][1] = y;
        }
        __syncthreads();
        x = y = 0.0;
#pragma unroll 4
        for (int w = 0; w < TV_WARPS; ++w) {
            x += sh.red[w][0];
            y += sh.red[w][1];
        }
    };
    // f(index, p logit, q logit) over the warp's elements, several loads in flight
    const float *lp = nullptr, *lq = nullptr;
    auto each = [&](auto f) {
#pragma unroll 1
        for (int i0 = w0 + lane * N; i0 < w1; i0 += 32 * N * 4) {
            float x[4][N], y[4][N];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + 32 * N * k;
                if (i < w1) {
                    tv_load<N>(x[k], lp + i);
                    if (DRAFT) tv_load<N>(y[k], lq + i);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + 32 * N * k;
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (i + j < w1) f(i + j, x[k][j], DRAFT ? y[k][j] : 0.f);
            }
        }
    };

    int cur = 0, count = 1;
    if (rank == 0)
        for (int i = tid; i < a.T; i += TV_THREADS) path[i] = i == 0 ? 0 : -1;
    for (;;) {
        lp = a.logits + ((size_t)b * a.T + cur) * a.ld;
        if (DRAFT) lq = a.draft + ((size_t)b * a.T + cur) * a.ld_draft;
        // the node's children and their logits
        if (tid < TREE_MAX_NODES) {
            const bool kid = tid > cur && tid < n && sh.par[tid] == cur;
            const unsigned m = __ballot_sync(0xFFFFFFFFu, kid);
            if (lane == 0) sh.kids[warp] = m;
            if (kid && !greedy) {
                const int x = sh.tok[tid];
                if (x >= 0 && x < V) sh.child[tid] = make_float2(lp[x], DRAFT ? lq[x] : 0.f);
            }
        }
        // pass 1: the maximum (temperature 0: with its first place)
        int best = 0;
        float mp = -INFINITY, mq = -INFINITY;
        if (greedy) {
            unsigned long long key = 0;
            each([&](int i, float x, float) {
                const unsigned long long k = argmax_key(x, (uint32_t)i);
                key = k > key ? k : key;
            });
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long k = __shfl_xor_sync(0xFFFFFFFFu, key, o);
                key = k > key ? k : key;
            }
            __syncthreads();
            if (lane == 0) sh.key[warp] = key;
            __syncthreads();
            for (int w = 0; w < TV_WARPS; ++w) key = sh.key[w] > key ? sh.key[w] : key;
            exchange(__longlong_as_double((long long)key), 0.0);
            for (int r = 0; r < C; ++r) {
                const unsigned long long k = (unsigned long long)__double_as_longlong(sh.ex[parity][r][0]);
                key = k > key ? k : key;
            }
            best = (int)key_index(key);
        } else {
            each([&](int, float x, float y) {
                mp = fmaxf(mp, x);
                if (DRAFT) mq = fmaxf(mq, y);
            });
            mp = warp_max(mp);
            if (DRAFT) mq = warp_max(mq);
            __syncthreads();
            if (lane == 0) {
                sh.red[warp][0] = (double)mp;
                sh.red[warp][1] = (double)mq;
            }
            __syncthreads();
            for (int w = 0; w < TV_WARPS; ++w) {
                mp = fmaxf(mp, (float)sh.red[w][0]);
                mq = fmaxf(mq, (float)sh.red[w][1]);
            }
            exchange((double)mp, (double)mq);
            for (int r = 0; r < C; ++r) {
                mp = fmaxf(mp, (float)sh.ex[parity][r][0]);
                mq = fmaxf(mq, (float)sh.ex[parity][r][1]);
            }
        }
        // pass 2: the sums
        double Sp = 0.0, Sq = 0.0;
        if (!greedy) {
            each([&](int, float x, float y) {
                Sp += (double)tv_weight(x, mp, a.inv_temp);
                if (DRAFT) Sq += (double)tv_weight(y, mq, a.inv_temp);
            });
            block_sum(Sp, Sq);
            exchange(Sp, Sq);
            Sp = Sq = 0.0;
            for (int r = 0; r < C; ++r) {
                Sp += sh.ex[parity][r][0];
                Sq += sh.ex[parity][r][1];
            }
        }
        const double ip = 1.0 / Sp;
        // the weight of a token in the residual p - c q, and the residual's sum over the cluster
        auto left = [&](float x, float y, double cq) {
            const double r = (double)tv_weight(x, mp, a.inv_temp) * ip;
            return DRAFT ? fmax(r - (double)tv_weight(y, mq, a.inv_temp) * cq, 0.0) : r;
        };
        double c = 0.0, W = 1.0;
        int n_gone = 0, taken = -1;
#pragma unroll 1
        for (int w = 0; w < (n + 31) / 32 && taken < 0; ++w)
#pragma unroll 1
            for (unsigned m = sh.kids[w]; m && taken < 0; m &= m - 1) {
                const int t = 32 * w + __ffs(m) - 1, x = sh.tok[t];
                if (x < 0 || x >= V) {
                    if (tid == 0 && rank == 0) atomicCAS(a.err, 0, ERR_BAD_TOKEN);
                    continue;
                }
                if (greedy) {
                    if (x == best) taken = t;
                    continue;
                }
                const float2 l = sh.child[t];
                const double ut = (double)sh.u[t];
                if (DRAFT) {
                    const double qx = (double)tv_weight(l.y, mq, a.inv_temp) / Sq;
                    if (ut * W * qx < left(l.x, l.y, c / Sq)) {
                        taken = t;
                    } else {
                        c += W;
                        const double cq = c / Sq;
                        double s = 0.0, z = 0.0;
                        each([&](int, float p, float q) { s += left(p, q, cq); });
                        block_sum(s, z);
                        exchange(s, 0.0);
                        W = 0.0;
                        for (int r = 0; r < C; ++r) W += sh.ex[parity][r][0];
                        if (!(W > 0.0)) {
                            c = 0.0;
                            W = 1.0;
                        }
                    }
                } else {
                    const bool out = __syncthreads_or(tid < n_gone && sh.gone[tid] == x);
                    const double r = out ? 0.0 : left(l.x, 0.f, 0.0);
                    if (ut * W < r) {
                        taken = t;
                    } else if (!out) {
                        W -= r;
                        if (tid == 0) {
                            sh.gone[n_gone] = x;
                            if (x >= s0 && x < s1) out_bits[(x - s0) >> 5] |= 1u << ((x - s0) & 31);
                        }
                        ++n_gone;
                        __syncthreads();
                    }
                }
            }
        if (taken >= 0) {
            if (tid == 0) {
                if (rank == 0) path[count] = taken;
                if (!DRAFT)
                    for (int g = 0; g < n_gone; ++g)
                        if (sh.gone[g] >= s0 && sh.gone[g] < s1) out_bits[(sh.gone[g] - s0) >> 5] = 0;
            }
            ++count;
            cur = taken;
            __syncthreads();
            continue;
        }
        // no child: the next token
        if (rank == 0 && tid == 0) a.n_path[b] = count;
        if (greedy) {
            if (rank == 0 && tid == 0) a.next[b] = best;
            return;
        }
        const double cq = DRAFT ? c / Sq : 0.0;
        auto rest = [&](int i, float p, float q) -> double {
            if (!DRAFT && n_gone && (out_bits[(i - s0) >> 5] >> ((i - s0) & 31) & 1)) return 0.0;
            return left(p, q, cq);
        };
        double mine = 0.0;
        each([&](int i, float p, float q) { mine += rest(i, p, q); });
        mine = warp_sum_d(mine);
        __syncthreads();
        if (lane == 0) sh.red[warp][0] = mine;
        __syncthreads();
        double sum = 0.0;
        for (int w = 0; w < TV_WARPS; ++w) sum += sh.red[w][0];
        exchange(sum, 0.0);
        double total = 0.0;
        for (int r = 0; r < C; ++r) total += sh.ex[parity][r][0];
        const double lim = (double)sh.u[0] * total;
        // the CTA, then the warp, whose part holds the limit (the last one with mass if rounding leaves none)
        double before = 0.0, at = 0.0;
        int cta = -1;
        for (int r = 0; r < C; ++r) {
            const double v = sh.ex[parity][r][0];
            if (v > 0.0) {
                cta = r;
                at = before;
                if (before + v > lim) break;
            }
            before += v;
        }
        if (cta < 0) {  // a row without mass
            if (rank == 0 && tid == 0) a.next[b] = 0;
            return;
        }
        if (cta != rank) return;
        before = at;
        int hit = -1;
        for (int w = 0; w < TV_WARPS; ++w) {
            const double v = sh.red[w][0];
            if (v > 0.0) {
                hit = w;
                at = before;
                if (before + v > lim) break;
            }
            before += v;
        }
        if (warp != hit) return;
        // 32 elements at a time: their prefix sums, the first that exceeds the limit
        int last = -1;
        for (int i0 = w0; i0 < w1; i0 += 32) {
            const int i = i0 + lane;
            const double r = i < w1 ? rest(i, lp[i], DRAFT ? lq[i] : 0.f) : 0.0;
            double inc = r;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                if (lane >= o) inc += v;
            }
            const unsigned over = __ballot_sync(0xFFFFFFFFu, r > 0.0 && at + inc > lim), some = __ballot_sync(0xFFFFFFFFu, r > 0.0);
            if (over) {
                if (lane == 0) a.next[b] = i0 + __ffs(over) - 1;
                return;
            }
            if (some) last = i0 + 31 - __clz(some);
            at += __shfl_sync(0xFFFFFFFFu, inc, 31);
        }
        if (lane == 0) a.next[b] = last;
        return;
    }
}

size_t tree_verify_ws_bytes(int, int, int) { return 256; }

template <int N, bool DRAFT>
static cudaError_t verify_launch(const TreeVerifyArgs& a, int C, cudaStream_t st) {
    auto fn = tf_tree_verify_kernel<N, DRAFT>;
    // slices of whole warps' pieces, pieces of whole vectors of 32 lanes
    const int unit = 32 * N, piece = ((a.V + C * TV_WARPS - 1) / (C * TV_WARPS) + unit - 1) / unit * unit, slice = piece * TV_WARPS;
    const size_t smem = DRAFT ? 0 : (size_t)(slice + 31) / 32 * 4;
    static std::atomic<bool> ready[64] = {};  // set once per device; twice is harmless
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (!ready[dev]) {
        cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        ready[dev].store(true);
    }
    if (smem > 100 * 1024) return cudaErrorInvalidValue;
    if (smem > 40 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.B * C));
    cfg.blockDim = dim3(TV_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, a, slice, piece);
}

cudaError_t tree_verify_launch(const TreeVerifyArgs& a, cudaStream_t st) {
    // CTAs per sequence: up to 16 while the batch leaves SMs free, so that two CTAs per SM hold it
    int C = TV_MAX_CLUSTER;
    while (C > 1 && (long long)a.B * C > 296) C /= 2;
    const bool vec = a.ld % 4 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 &&
                     (!a.draft || (a.ld_draft % 4 == 0 && (reinterpret_cast<uintptr_t>(a.draft) & 15) == 0)) && a.V % 4 == 0;
    if (a.draft) return vec ? verify_launch<4, true>(a, C, st) : verify_launch<1, true>(a, C, st);
    return vec ? verify_launch<4, false>(a, C, st) : verify_launch<1, false>(a, C, st);
}

}  // namespace tfb
