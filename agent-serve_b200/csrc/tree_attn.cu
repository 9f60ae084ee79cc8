// Attention of a tree of drafted tokens over the KV cache.
//
// Row (b, t, h): s_j = q . k_j / sqrt(hd) over the visible positions j, p_j = exp(s_j - max s),
// out = sum p_j v_j / sum p_j; a row that sees nothing is zero.
#include "tree.cuh"

namespace tfb {

constexpr int TA_THREADS = 128;

__global__ void __launch_bounds__(TA_THREADS) tf_tree_attn_kernel(const TreeAttnArgs a) {
    __shared__ float qs[AT_MAX_HD], sc[TA_THREADS], red[TA_THREADS / 32];
    const int h = blockIdx.x, t = blockIdx.y, b = blockIdx.z;
    const int tid = threadIdx.x, hd = a.hd, kvh = h / (a.n_head / a.n_kv);
    const size_t row = (size_t)b * a.T + t;
    float* out = a.out + row * a.ld_out + (size_t)h * hd;
    const int slot = a.slots ? a.slots[b] : b, n_ctx = a.n_ctx[b];
    const int n_node = a.n_node ? min(a.n_node[b], a.T) : a.T;
    const bool bad = slot < 0 || slot >= a.n_slots || n_ctx < 0 || n_node < 0 || n_ctx > a.cap - n_node;
    if (bad && tid == 0) atomicCAS(a.err, 0, ERR_POS);
    if (bad || t >= n_node) {
        for (int d = tid; d < hd; d += TA_THREADS) out[d] = 0.f;
        return;
    }
    for (int d = tid; d < hd; d += TA_THREADS) qs[d] = a.q[row * a.ld_q + (size_t)h * hd + d];
    const unsigned long long* mw = a.mask ? a.mask + row * ((a.T + 63) / 64) : nullptr;
    const long long base = (long long)slot * a.slot_stride + (long long)kvh * a.cap * hd;
    const float scale = 1.0f / sqrtf((float)hd);
    float mx = -INFINITY, den = 0.f, acc = 0.f;  // acc: dim tid
    __syncthreads();
    for (int p0 = 0; p0 < n_ctx + n_node; p0 += TA_THREADS) {
        const int p = p0 + tid, j = p - n_ctx;
        bool vis = p < n_ctx + n_node;
        if (vis && j >= 0) vis = mw ? (mw[j >> 6] >> (j & 63)) & 1 : j <= t;
        float s = -INFINITY;
        if (vis) {
            s = 0.f;
            for (int d = 0; d < hd; ++d) s = fmaf(qs[d], kv_load(a.kc, base + (long long)p * hd + d, a.kv_type), s);
            s *= scale;
        }
        float m = warp_max(s);
        if ((tid & 31) == 0) red[tid >> 5] = m;
        __syncthreads();
        m = mx;
        for (int w = 0; w < TA_THREADS / 32; ++w) m = fmaxf(m, red[w]);
        sc[tid] = vis ? expf(s - m) : -1.f;  // -1: masked, its value is not read
        __syncthreads();
        if (m > -INFINITY) {
            const float al = expf(mx - m);
            den *= al;
            acc *= al;
        }
        mx = m;
        for (int i = 0; i < TA_THREADS; ++i) {
            const float e = sc[i];
            if (e == -1.f) continue;
            den += e;
            if (tid < hd) acc = fmaf(e, kv_load(a.vc, base + (long long)(p0 + i) * hd + tid, a.kv_type), acc);
        }
        __syncthreads();
    }
    if (tid < hd) out[tid] = den == 0.f ? 0.f : acc / den;
}

size_t tree_attn_ws_bytes(int, int, int, int, int) { return 256; }

cudaError_t tree_attn_launch(const TreeAttnArgs& a, cudaStream_t st, bool) {
    tf_tree_attn_kernel<<<dim3(a.n_head, a.T, a.B), TA_THREADS, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace tfb
