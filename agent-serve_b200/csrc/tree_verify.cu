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
// exponentials are 32-bit, every sum and residual is held in 64 bits.
#include "tree.cuh"

namespace tfb {

constexpr int TV_THREADS = 1024;

// exp(l / temp - max): 1 at the maximum itself (also an infinite one); a NaN logit weighs nothing
__device__ __forceinline__ float tv_weight(float l, float mx, float inv_temp) {
    return l == mx ? 1.f : (l != l ? 0.f : expf(__fmul_rn(__fsub_rn(l, mx), inv_temp)));
}

__device__ __forceinline__ double tv_sum(double v, double* red) {
    v = warp_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0;
    for (int w = 0; w < TV_THREADS / 32; ++w) s += red[w];
    return s;
}

__global__ void __launch_bounds__(TV_THREADS) tf_tree_verify_kernel(const TreeVerifyArgs a) {
    __shared__ double red[TV_THREADS / 32];
    __shared__ double scan[TV_THREADS];
    __shared__ unsigned long long keys[TV_THREADS / 32];
    __shared__ int gone[TREE_MAX_NODES];
    __shared__ int pick_s;
    const int b = blockIdx.x, tid = threadIdx.x, V = a.V;
    const int n = a.n_node ? min(max(a.n_node[b], 0), a.T) : a.T;
    int* path = a.path + (size_t)b * a.T;
    for (int i = tid; i < a.T; i += TV_THREADS) path[i] = -1;
    __syncthreads();
    if (n == 0) {
        if (tid == 0) {
            a.n_path[b] = 0;
            a.next[b] = -1;
        }
        return;
    }
    const int *tok = a.tokens + (size_t)b * a.T, *par = a.parents + (size_t)b * a.T;
    const float* u = a.u + (size_t)b * a.T;
    int cur = 0, count = 1, n_gone = 0;
    double c = 0.0, W = 1.0;
    for (;;) {
        const float* lp = a.logits + ((size_t)b * a.T + cur) * a.ld;
        const float* lq = a.draft ? a.draft + ((size_t)b * a.T + cur) * a.ld_draft : nullptr;
        // the row's maximum (its first place) and sums
        unsigned long long key = 0, kq = 0;
        for (int i = tid; i < V; i += TV_THREADS) {
            // sampling: a NaN logit weighs nothing; greedy: argmax_key's own rule
            const unsigned long long k = lp[i] != lp[i] && a.inv_temp > 0.f ? 0ull : argmax_key(lp[i], (uint32_t)i);
            key = k > key ? k : key;
            if (lq) {
                const unsigned long long k2 = lq[i] != lq[i] ? 0ull : argmax_key(lq[i], (uint32_t)i);
                kq = k2 > kq ? k2 : kq;
            }
        }
        auto block_max = [&](unsigned long long k) {
            for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long w = __shfl_xor_sync(0xFFFFFFFFu, k, o);
                k = w > k ? w : k;
            }
            __syncthreads();
            if ((tid & 31) == 0) keys[tid >> 5] = k;
            __syncthreads();
            for (int w = 0; w < TV_THREADS / 32; ++w) k = keys[w] > k ? keys[w] : k;
            return k;
        };
        key = block_max(key);
        const int best = key ? (int)key_index(key) : 0;
        const float mp = key ? lp[best] : -INFINITY;
        float mq = 0.f;
        double Sp = 1.0, Sq = 1.0;
        if (a.inv_temp > 0.f) {
            double s = 0.0;
            for (int i = tid; i < V; i += TV_THREADS) s += (double)tv_weight(lp[i], mp, a.inv_temp);
            Sp = tv_sum(s, red);
            if (lq) {
                kq = block_max(kq);
                mq = kq ? lq[key_index(kq)] : -INFINITY;
                s = 0.0;
                for (int i = tid; i < V; i += TV_THREADS) s += (double)tv_weight(lq[i], mq, a.inv_temp);
                Sq = tv_sum(s, red);
            }
        }
        auto left = [&](int i, double cc) {  // the residual's weight of token i
            double r = (double)tv_weight(lp[i], mp, a.inv_temp) / Sp;
            if (lq) r = fmax(r - (double)tv_weight(lq[i], mq, a.inv_temp) * (cc / Sq), 0.0);
            for (int g = 0; g < n_gone; ++g)
                if (gone[g] == i) r = 0.0;
            return r;
        };
        int taken = -1;
        for (int t = cur + 1; t < n && taken < 0; ++t) {
            if (par[t] != cur) continue;
            const int x = tok[t];
            if (x < 0 || x >= V) {
                if (tid == 0) atomicCAS(a.err, 0, ERR_BAD_TOKEN);
                continue;
            }
            if (a.inv_temp == 0.f) {
                if (x == best) taken = t;
                continue;
            }
            const double r = left(x, c), ut = (double)u[t];
            if (lq) {
                const double qx = (double)tv_weight(lq[x], mq, a.inv_temp) / Sq;
                if (ut * W * qx < r) {
                    taken = t;
                } else {
                    c += W;
                    double s = 0.0;
                    for (int i = tid; i < V; i += TV_THREADS) s += left(i, c);
                    W = tv_sum(s, red);
                    if (!(W > 0.0)) {
                        c = 0.0;
                        W = 1.0;
                    }
                }
            } else if (ut * W < r) {
                taken = t;
            } else {
                W -= r;
                __syncthreads();
                if (tid == 0) gone[n_gone] = x;
                __syncthreads();
                ++n_gone;
            }
        }
        if (taken >= 0) {
            if (tid == 0) path[count] = taken;
            ++count;
            cur = taken;
            c = 0.0;
            W = 1.0;
            n_gone = 0;
            continue;
        }
        // the next token
        if (tid == 0) {
            path[0] = 0;
            a.n_path[b] = count;
            pick_s = best;
        }
        if (a.inv_temp > 0.f) {
            const int per = (V + TV_THREADS - 1) / TV_THREADS, i0 = min(V, tid * per), i1 = min(V, i0 + per);
            double s = 0.0;
            for (int i = i0; i < i1; ++i) s += left(i, c);
            scan[tid] = s;
            __syncthreads();
            double before = 0.0, total = 0.0;
            for (int w = 0; w < TV_THREADS; ++w) {
                if (w == tid) before = total;
                total += scan[w];
            }
            const double lim = (double)u[0] * total;
            if (before <= lim && before + s > lim) {
                for (int i = i0; i < i1; ++i) {
                    before += left(i, c);
                    if (before > lim) {
                        pick_s = i;
                        break;
                    }
                }
            }
        }
        __syncthreads();
        if (tid == 0) a.next[b] = pick_s;
        return;
    }
}

size_t tree_verify_ws_bytes(int, int, int) { return 256; }

cudaError_t tree_verify_launch(const TreeVerifyArgs& a, cudaStream_t st) {
    tf_tree_verify_kernel<<<a.B, TV_THREADS, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace tfb
