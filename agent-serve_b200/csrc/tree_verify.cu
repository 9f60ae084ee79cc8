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
// contiguous slice of the vocabulary, each warp a contiguous piece of the slice, which it brings
// into shared memory by a bulk copy of its own.  A visited row takes two passes (maximum, then
// weights, in place, and sums), a rejection with a draft distribution and the final pick one more
// each over the weights.  After a pass each CTA joins its warps' values and writes the result into
// every CTA's shared memory; behind one cluster barrier every warp joins those in the same order:
// all CTAs hold the same sums and take the same decisions.  A walk is a chain of such rows, so its
// latency bounds it: when all rows of all trees fit on the GPU at once, and there is a draft
// distribution, one cluster per row finds every row's maximum and sum first (ROWS), and the walk
// behind it takes passes for rejections and picks only.
//
// A visited row takes about 14000 cycles of a draft walk (load 3000, maximum 1400, exchange 3200,
// weights 4100, exchange and division 2400).  16 CTAs per sequence: the two rows of 128000 tokens
// are then 64 KB per CTA, two CTAs per SM, and 18 sequences are resident at once.  Device time,
// 128256 tokens: a chain of 6 with draft 18 us, a greedy tree of 32 11.8 us; 151936 tokens: 32
// chains of 8 with draft 116 us (143 MB read: 1.2 TB/s; two waves of sequences), 16 trees of 25
// without draft 32 us.
#include <cooperative_groups.h>

#include <atomic>

#include "tree.cuh"

namespace cg = cooperative_groups;

namespace tfb {

constexpr int TV_THREADS = 512;
constexpr int TV_WARPS = TV_THREADS / 32;
constexpr int TV_CLUSTER = 16;
static_assert(TV_WARPS == 16 && TV_CLUSTER == 16, "values are joined and searched sixteen at a time");

struct TvStats {                       // of a node's rows: maxima, and 1 / sum of the weights relative to them
    double ip, iq;
    float mp, mq;
};
// Rows whose clusters fit the GPU at once (16 CTAs each, two per SM).  With a draft distribution their
// statistics are found ahead of the walk; mean over 16 chains of 128256 tokens without / with it:
// 2 nodes (1.8 rows visited) 15.9 / 16.2 us, 6 nodes (3.3) 26.3 / 20.1, 12 nodes (4.2) 32.6 / 24.7, 18
// nodes 33.1 / 30.5; 32 nodes in two waves 33 / 50.  Without a distribution, or greedy, a row of the walk
// is cheaper and fewer are visited: 12 nodes 11.4 / 15.1 and 10.5 / 10.1, 18 nodes 11.4 / 17.8 and
// 10.4 / 12.5, so those walk at once.
constexpr int TV_MAX_STATS = 18;

struct TvShared {
    double2 warps[2][TV_WARPS];        // this CTA's values, one per warp, of the last two exchanges
    double2 ex[2][TV_CLUSTER];     // every CTA's
    uint64_t landed[TV_WARPS];
    int par[TREE_MAX_NODES], tok[TREE_MAX_NODES];
    float u[TREE_MAX_NODES];
    float2 child[TREE_MAX_NODES];      // each node's logits in its parent's rows: target, draft
    TvStats st[TV_MAX_STATS];
    unsigned kids[TREE_MAX_NODES / 32];
    int gone[TREE_MAX_NODES];          // tokens taken out of p at this node
};

struct TvPlan {
    int slice, piece;                  // elements of a CTA, of a warp (multiples of 4)
    int stats;                         // walk: the rows' statistics are in the workspace
};

// A row's softmax weights relative to its maximum: exp((l - max) / temp), 1 at an infinite
// maximum, 0 for a NaN logit.
struct TvRow {
    float mx, inv_temp;
    bool inf;
    __device__ __forceinline__ float finite_weight(float l) const {
        return fmaxf(expf(__fmul_rn(__fsub_rn(l, mx), inv_temp)), 0.f);
    }
    __device__ __forceinline__ float weight(float l) const { return inf ? (l == mx ? 1.f : 0.f) : finite_weight(l); }
};
__device__ __forceinline__ TvRow tv_row(float mx, float inv_temp) { return TvRow{mx, inv_temp, !(fabsf(mx) < INFINITY)}; }

// A weight in 64 bits by integer instructions (a conversion shares the exponentials' pipe, which
// bounds the pass): exact from 2^-126 on, off by 2^-127 at most below it and at zero, which no sum
// of weights sees: its largest term is 1.  (Not for residuals: there a zero has to be one.)
__device__ __forceinline__ double weight_wide(float x) {
    const unsigned long long b = (unsigned long long)__float_as_uint(x) * (1u << 29);
    return __hiloint2double((int)(b >> 32) + (896 << 20), (int)b);
}

// A warp's piece of logits into weights, in place, and their sums; elements behind its end become
// weights of zero (FULL: pieces end at a multiple of four).  One copy of the code: it is fetched
// anew by each CTA.
template <bool DRAFT, bool FULL>
__device__ __noinline__ double2 tv_weights(float* rp, float* rq, int wn, TvRow P, TvRow Q) {
    double2 s = make_double2(0.0, 0.0);
    auto vec = [](float4 x, int k, const TvRow& R, double& sum, auto weight) {  // k: elements left
        x = make_float4(weight(R, x.x), FULL || k > 1 ? weight(R, x.y) : 0.f, FULL || k > 2 ? weight(R, x.z) : 0.f,
                        FULL || k > 3 ? weight(R, x.w) : 0.f);
        sum += (weight_wide(x.x) + weight_wide(x.y)) + (weight_wide(x.z) + weight_wide(x.w));
        return x;
    };
    auto pass = [&](auto weight) {
#pragma unroll 2
        for (int i = (threadIdx.x & 31) * 4; i < wn; i += 128) {
            const float4 x = *reinterpret_cast<const float4*>(rp + i);
            const float4 y = DRAFT ? *reinterpret_cast<const float4*>(rq + i) : x;
            *reinterpret_cast<float4*>(rp + i) = vec(x, wn - i, P, s.x, weight);
            if (DRAFT) *reinterpret_cast<float4*>(rq + i) = vec(y, wn - i, Q, s.y, weight);
        }
    };
    if (P.inf || (DRAFT && Q.inf)) pass([](const TvRow& R, float l) { return R.weight(l); });
    else pass([](const TvRow& R, float l) { return R.finite_weight(l); });
    __syncwarp();
    return make_double2(warp_sum_d(s.x), DRAFT ? warp_sum_d(s.y) : 0.0);
}

// the residual p - c q of weights x and y (ip = 1 / sum x, cq = c / sum y)
template <bool DRAFT>
__device__ __forceinline__ double tv_left(float x, float y, double ip, double cq) {
    const double r = (double)x * ip;
    return DRAFT ? fmax(r - (double)y * cq, 0.0) : r;
}
// its sum over a warp's piece
template <bool DRAFT>
__device__ __noinline__ double tv_rest(const float* rp, const float* rq, int wn, double ip, double cq) {
    double s = 0.0;
#pragma unroll 2
    for (int i = (threadIdx.x & 31) * 4; i < wn; i += 128) {
        const float4 x = *reinterpret_cast<const float4*>(rp + i);
        const float4 y = DRAFT ? *reinterpret_cast<const float4*>(rq + i) : x;
        s += (tv_left<DRAFT>(x.x, y.x, ip, cq) + tv_left<DRAFT>(x.y, y.y, ip, cq)) +
             (tv_left<DRAFT>(x.z, y.z, ip, cq) + tv_left<DRAFT>(x.w, y.w, ip, cq));
    }
    return warp_sum_d(s);
}

// VEC: rows are 16-byte aligned and V % 4 == 0 (bulk copies); ROWS: statistics of every node's rows,
// one cluster each, else the walk, one cluster per sequence
template <bool VEC, bool DRAFT, bool ROWS>
__global__ void __launch_bounds__(TV_THREADS, 2)
    tf_tree_verify_kernel(const __grid_constant__ TreeVerifyArgs a, const __grid_constant__ TvPlan pl) {
    extern __shared__ __align__(16) float rows[];  // the slice of the target's row, of the draft's
    __shared__ __align__(16) TvShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    constexpr int C = TV_CLUSTER;
    const int rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = a.V;
    const int b = ROWS ? blockIdx.x / C / a.T : blockIdx.x / C;
    pdl_trigger();
    pdl_wait();
    const int n = a.n_node ? min(max(a.n_node[b], 0), a.T) : a.T;
    int cur = ROWS ? blockIdx.x / C % a.T : 0;
    if (ROWS && cur >= n) return;
    int* path = a.path + (size_t)b * a.T;
    if (!ROWS && n == 0) {
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
    TvStats* stats = static_cast<TvStats*>(a.ws);
    if (!ROWS) {
        if (tid < n) {
            sh.par[tid] = a.parents[(size_t)b * a.T + tid];
            sh.tok[tid] = a.tokens[(size_t)b * a.T + tid];
            sh.u[tid] = greedy ? 0.f : a.u[(size_t)b * a.T + tid];
            const int x = sh.tok[tid], p = sh.par[tid];
            if (!greedy && x >= 0 && x < V && p >= 0 && p < tid) {
                const size_t r = (size_t)b * a.T + p;
                sh.child[tid] = make_float2(a.logits[r * a.ld + x], DRAFT ? a.draft[r * a.ld_draft + x] : 0.f);
            }
            if (pl.stats) sh.st[tid] = stats[(size_t)b * a.T + tid];
        }
        if (rank == 0 && tid < a.T) path[tid] = tid == 0 ? 0 : -1;
    }
    if (tid < TV_WARPS) mbar_init(&sh.landed[tid], 1);
    if (tid == 0) mbar_fence_init();
    cluster.sync();  // (a CTA's shared memory is written by others only once it runs)

    // this warp's elements [w0, w1) of the row, at rp and rq
    const int s0 = min(V, rank * pl.slice), s1 = min(V, s0 + pl.slice);
    const int w0 = min(s1, s0 + warp * pl.piece), w1 = min(s1, w0 + pl.piece), wn = w1 - w0;
    float* const rp = rows + warp * pl.piece;
    float* const rq = rp + pl.slice;
    int parity = 0, loads = 0;
    const float *lp = nullptr, *lq = nullptr;
    auto load_begin = [&]() {
        if (VEC) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0 && wn) {
                mbar_expect_tx(&sh.landed[warp], (uint32_t)wn * (DRAFT ? 8u : 4u));
                bulk_g2s(rp, lp + w0, (uint32_t)wn * 4u, &sh.landed[warp]);
                if (DRAFT) bulk_g2s(rq, lq + w0, (uint32_t)wn * 4u, &sh.landed[warp]);
            }
        }
    };
    auto load_end = [&]() {
        if (VEC) {
            if (wn) mbar_wait(&sh.landed[warp], loads & 1, a.err, ERR_WAIT_FULL, nullptr);
            ++loads;
        } else {
#pragma unroll 4
            for (int i = lane; i < wn; i += 32) {
                rp[i] = lp[w0 + i];
                if (DRAFT) rq[i] = lq[w0 + i];
            }
        }
        __syncwarp();
    };
    // f(p, q, index) on the lane's vectors of the piece (its last one may reach behind the end)
    auto each = [&](auto f) {
#pragma unroll 2
        for (int i = lane * 4; i < wn; i += 128) {
            float4 x = *reinterpret_cast<const float4*>(rp + i), y = x;
            if (DRAFT) y = *reinterpret_cast<const float4*>(rq + i);
            f(x, y, i);
        }
        __syncwarp();
    };
    // Joins one value pair per warp over the cluster, in the same order in every warp; on the way the
    // warps' pairs stay in sh.warps[parity], the CTAs' in sh.ex[parity].
    auto exchange = [&](double x, double y, auto join) {
        parity ^= 1;
        auto join16 = [&](double2 v) {
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) {
                const double2 z = make_double2(__shfl_xor_sync(0xFFFFFFFFu, v.x, o), DRAFT ? __shfl_xor_sync(0xFFFFFFFFu, v.y, o) : 0.0);
                v = make_double2(join(v.x, z.x), DRAFT ? join(v.y, z.y) : 0.0);
            }
            return v;
        };
        if (lane == 0) sh.warps[parity][warp] = make_double2(x, y);
        __syncthreads();
        if (warp == 0) {
            const double2 v = join16(sh.warps[parity][lane % TV_WARPS]);
            if (lane < TV_CLUSTER) *cluster.map_shared_rank(&sh.ex[parity][rank], lane) = v;
        }
        cluster.sync();
        return join16(sh.ex[parity][lane % TV_CLUSTER]);
    };
    auto add = [](double x, double y) { return x + y; };

    int count = 1;
    for (;;) {
        lp = a.logits + ((size_t)b * a.T + cur) * a.ld;
        if (DRAFT) lq = a.draft + ((size_t)b * a.T + cur) * a.ld_draft;
        if (ROWS || !pl.stats) load_begin();
        // the node's children (read after the next barrier)
        if (!ROWS && tid < TREE_MAX_NODES) {
            const bool kid = tid > cur && tid < n && sh.par[tid] == cur;
            const unsigned m = __ballot_sync(0xFFFFFFFFu, kid);
            if (lane == 0) sh.kids[warp] = m;
        }
        int best = 0;
        TvRow P, Q;
        double ip = 0.0, iq = 0.0;
        bool weights = false;  // the slice holds weights
        if (!ROWS && pl.stats) {
            P = tv_row(sh.st[cur].mp, a.inv_temp);
            Q = tv_row(sh.st[cur].mq, a.inv_temp);
            ip = sh.st[cur].ip;
            iq = sh.st[cur].iq;
            __syncthreads();
        } else {
            load_end();
            if (!DRAFT && greedy) {  // the maximum with its first place
                unsigned long long key = 0;
                each([&](float4 x, float4, int i) {
                    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const unsigned long long k = i + e < wn ? argmax_key(v[e], (uint32_t)(w0 + i + e)) : 0ull;
                        key = k > key ? k : key;
                    }
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const unsigned long long k = __shfl_xor_sync(0xFFFFFFFFu, key, o);
                    key = k > key ? k : key;
                }
                key = (unsigned long long)__double_as_longlong(
                    exchange(__longlong_as_double((long long)key), 0.0, [](double x, double y) {
                        return (unsigned long long)__double_as_longlong(x) > (unsigned long long)__double_as_longlong(y) ? x : y;
                    }).x);
                best = (int)key_index(key);
            } else {
                float mp = -INFINITY, mq = -INFINITY;
                each([&](float4 x, float4 y, int i) {
                    const int k = wn - i;
                    mp = fmaxf(mp, x.x);
                    if (k > 1) mp = fmaxf(mp, x.y);
                    if (k > 2) mp = fmaxf(mp, x.z);
                    if (k > 3) mp = fmaxf(mp, x.w);
                    if (DRAFT) {
                        mq = fmaxf(mq, y.x);
                        if (k > 1) mq = fmaxf(mq, y.y);
                        if (k > 2) mq = fmaxf(mq, y.z);
                        if (k > 3) mq = fmaxf(mq, y.w);
                    }
                });
                mp = warp_max(mp);
                if (DRAFT) mq = warp_max(mq);
                const double2 m = exchange((double)mp, (double)mq, [](double x, double y) { return x > y ? x : y; });
                P = tv_row((float)m.x, a.inv_temp);
                Q = DRAFT ? tv_row((float)m.y, a.inv_temp) : P;
                const double2 ws = tv_weights<DRAFT, VEC>(rp, rq, wn, P, Q);
                weights = true;
                const double2 S = exchange(ws.x, ws.y, add);
                ip = 1.0 / S.x;
                if (DRAFT) iq = 1.0 / S.y;
            }
        }
        if (ROWS) {
            if (rank == 0 && tid == 0)
                stats[(size_t)b * a.T + cur] = TvStats{ip, iq, P.mx, Q.mx};
            return;
        }
        auto need_weights = [&]() {
            if (weights) return;
            load_begin();
            load_end();
            tv_weights<DRAFT, VEC>(rp, rq, wn, P, Q);
            weights = true;
        };
        double c = 0.0, W = 1.0;
        int n_gone = 0, taken = -1;
#pragma unroll 1
        for (int t = cur + 1; t < n && taken < 0; ++t) {
            // the next child from t on
            const unsigned m = sh.kids[t >> 5] >> (t & 31);
            if (!m) {
                t |= 31;
                continue;
            }
            t += __ffs(m) - 1;
            const int x = sh.tok[t];
            if (x < 0 || x >= V) {
                if (tid == 0 && rank == 0) atomicCAS(a.err, 0, ERR_BAD_TOKEN);
                continue;
            }
            if (!DRAFT && greedy) {
                if (x == best) taken = t;
                continue;
            }
            const float2 l = sh.child[t];
            const float xw = P.weight(l.x);
            const double ut = (double)sh.u[t];
            if (DRAFT) {
                const float yw = Q.weight(l.y);
                if (ut * W * ((double)yw * iq) < tv_left<DRAFT>(xw, yw, ip, c * iq)) {
                    taken = t;
                } else {
                    need_weights();
                    c += W;
                    W = exchange(tv_rest<DRAFT>(rp, rq, wn, ip, c * iq), 0.0, add).x;
                    if (!(W > 0.0)) {
                        c = 0.0;
                        W = 1.0;
                    }
                }
            } else {
                const bool out = __syncthreads_or(tid < n_gone && sh.gone[tid] == x);
                const double r = out ? 0.0 : tv_left<DRAFT>(xw, 0.f, ip, 0.0);
                if (ut * W < r) {
                    taken = t;
                } else if (!out) {
                    W -= r;
                    if (tid == 0) {
                        sh.gone[n_gone] = x;
                    }
                    ++n_gone;
                    __syncthreads();
                }
            }
        }
        if (taken >= 0) {
            if (rank == 0 && tid == 0) path[count] = taken;
            ++count;
            cur = taken;
            __syncthreads();  // the children's table is read
            continue;
        }
        // no child: the next token
        if (rank == 0 && tid == 0) a.n_path[b] = count;
        if (!DRAFT && greedy) {
            if (rank == 0 && tid == 0) a.next[b] = best;
            return;
        }
        need_weights();
        const double cq = c * iq;
        if (!DRAFT && n_gone) {  // tokens out of p weigh nothing
            for (int g = lane; g < n_gone; g += 32) {
                const int x = sh.gone[g];
                if (x >= w0 && x < w1) rp[x - w0] = 0.f;
            }
            __syncwarp();
        }
        const double lim = (double)sh.u[0] * exchange(tv_rest<DRAFT>(rp, rq, wn, ip, cq), 0.0, add).x;
        // Of 16 masses, lane i (and i + 16) holding the i-th, the first whose running sum passes the
        // limit, or the last with mass if rounding leaves none; `at` moves up to its start.  -1: no mass.
        double at = 0.0;
        auto find16 = [&](double v) {
            double run = v;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                const double z = __shfl_up_sync(0xFFFFFFFFu, run, o, 16);
                if (lane % 16 >= o) run += z;
            }
            const unsigned some = __ballot_sync(0xFFFFFFFFu, v > 0.0) & 0xFFFFu;
            const unsigned over = __ballot_sync(0xFFFFFFFFu, v > 0.0 && at + run > lim) & 0xFFFFu;
            if (!some) return -1;
            const int src = over ? __ffs(over) - 1 : 31 - __clz(some);
            at += __shfl_sync(0xFFFFFFFFu, run - v, src);
            return src;
        };
        const int hit = find16(sh.ex[parity][lane % TV_CLUSTER].x);
        if (hit < 0) {  // a row without mass
            if (rank == 0 && tid == 0) a.next[b] = 0;
            return;
        }
        if (hit != rank || find16(sh.warps[parity][lane % TV_WARPS].x) != warp) return;
        // 128 elements at a time, four per lane: prefix sums, the first that passes the limit
        int last = -1;
#pragma unroll 1
        for (int i0 = 0; i0 < wn; i0 += 128) {
            const int i = i0 + 4 * lane;
            double r[4] = {0.0, 0.0, 0.0, 0.0}, sum = 0.0;
            if (i < wn) {
                const float4 x = *reinterpret_cast<const float4*>(rp + i), y = DRAFT ? *reinterpret_cast<const float4*>(rq + i) : x;
                r[0] = tv_left<DRAFT>(x.x, y.x, ip, cq), r[1] = tv_left<DRAFT>(x.y, y.y, ip, cq);
                r[2] = tv_left<DRAFT>(x.z, y.z, ip, cq), r[3] = tv_left<DRAFT>(x.w, y.w, ip, cq);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) sum += r[k];
            double s = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double z = __shfl_up_sync(0xFFFFFFFFu, s, o);
                if (lane >= o) s += z;
            }
            double run = at + (s - sum);
            int first = -1, pos = -1;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                run += r[k];
                if (r[k] > 0.0) {
                    pos = i + k;
                    if (first < 0 && run > lim) first = i + k;
                }
            }
            const unsigned m = __ballot_sync(0xFFFFFFFFu, first >= 0), w = __ballot_sync(0xFFFFFFFFu, pos >= 0);
            if (m) {
                if (lane == __ffs(m) - 1) a.next[b] = w0 + first;
                return;
            }
            if (w) last = w0 + __shfl_sync(0xFFFFFFFFu, pos, 31 - __clz(w));
            at += __shfl_sync(0xFFFFFFFFu, s, 31);
        }
        if (lane == 0) a.next[b] = last;
        return;
    }
}

size_t tree_verify_ws_bytes(int B, int T, int) { return 256 + (size_t)B * T * sizeof(TvStats); }

int tree_verify_max_vocab(bool draft) { return (TV_CLUSTER * (200 * 1024 / (draft ? 8 : 4))) / 1024 * 1024; }

template <bool VEC, bool DRAFT, bool ROWS>
static cudaError_t verify_launch(const TreeVerifyArgs& a, TvPlan pl, cudaStream_t st, bool pdl) {
    auto fn = tf_tree_verify_kernel<VEC, DRAFT, ROWS>;
    constexpr int C = TV_CLUSTER;
    pl.piece = ((a.V + C * TV_WARPS - 1) / (C * TV_WARPS) + 3) / 4 * 4;
    pl.slice = pl.piece * TV_WARPS;
    const size_t smem = (size_t)pl.slice * (DRAFT ? 8 : 4);
    static std::atomic<bool> ready[64] = {};  // set once per device; twice is harmless
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (!ready[dev]) {
        cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 208 * 1024);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return e;
        ready[dev].store(true);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((ROWS ? a.B * a.T : a.B) * C));
    cfg.blockDim = dim3(TV_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, fn, a, pl);
}

template <bool VEC, bool DRAFT>
static cudaError_t verify_run(const TreeVerifyArgs& a, cudaStream_t st) {
    TvPlan pl = {};
    pl.stats = DRAFT && a.T > 1 && a.B * a.T <= TV_MAX_STATS;
    if constexpr (DRAFT) {
        if (pl.stats) {
            const cudaError_t e = verify_launch<VEC, DRAFT, true>(a, pl, st, false);
            if (e != cudaSuccess) return e;
        }
    }
    return verify_launch<VEC, DRAFT, false>(a, pl, st, pl.stats);
}

cudaError_t tree_verify_launch(const TreeVerifyArgs& a, cudaStream_t st) {
    const bool vec = a.ld % 4 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 &&
                     (!a.draft || (a.ld_draft % 4 == 0 && (reinterpret_cast<uintptr_t>(a.draft) & 15) == 0)) && a.V % 4 == 0;
    if (a.draft) return vec ? verify_run<true, true>(a, st) : verify_run<false, true>(a, st);
    return vec ? verify_run<true, false>(a, st) : verify_run<false, false>(a, st);
}

}  // namespace tfb
