// Commit of an accepted path of drafted nodes: cache row n_ctx + i <- row n_ctx + path[i], in
// place, for K and V of every layer and kv head, so that the path's rows follow the committed
// context without gaps.
//
// One warp per (layer, sequence, kv head, K or V).  The path is strictly increasing, so
// path[i] >= i: taking the rows in ascending groups, each group loaded into registers before it
// is stored, never reads a row that an earlier group has overwritten.  Rows that stay where they
// are (the root's) are not moved.  Bound by latency (lengths and path, then a few rows of 128 to 512
// bytes per warp): 16 layers of 8 kv heads, one path of 5 rows 2.2 us; 28 layers of 2 kv heads of 128
// dims fp32, 64 paths of 7 rows 9.4 us (44 MB read and written: 4.7 TB/s).
#include "tree.cuh"

namespace tfb {

constexpr int KC_THREADS = 128;
constexpr int KC_VEC = 8;  // 16-byte vectors in flight per lane

__global__ void __launch_bounds__(KC_THREADS) tf_kv_commit_kernel(const KvCommitArgs a) {
    const int lane = threadIdx.x & 31;
    const unsigned unit = (unsigned)(((unsigned long long)blockIdx.x * KC_THREADS + threadIdx.x) >> 5);
    if (unit >= (unsigned)a.n_layer * a.B * a.n_kv * 2u) return;
    const int kv = (int)(unit & 1);                                  // layer, sequence, kv head, K / V
    const unsigned seq = (unit >> 1) / (unsigned)a.n_kv;
    const int h = (int)((unit >> 1) - seq * a.n_kv);
    const int layer = (int)(seq / (unsigned)a.B), b = (int)(seq - (unsigned)layer * a.B);
    const int slot = a.slots ? a.slots[b] : b, n_ctx = a.n_ctx[b], n = a.n_path[b];
    const int* path = a.path + (long long)b * a.ld_path;
    bool bad = slot < 0 || slot >= a.n_slots || n_ctx < 0 || n_ctx > a.cap || n < 0 || n > a.ld_path;
    if (!bad)
        for (int i = lane; i < n; i += 32) {
            const int p = path[i];
            bad |= p < i || p >= a.cap - n_ctx || (i > 0 && p <= path[i - 1]);
        }
    bad = __any_sync(0xFFFFFFFFu, bad);
    if (layer == 0 && kv == 0 && h == 0 && lane == 0) {
        if (bad) atomicCAS(a.err, 0, ERR_POS);
        if (a.n_new) a.n_new[b] = bad ? n_ctx : n_ctx + n;
    }
    if (bad || n == 0) return;
    const int vpr = a.hd * a.elem_bytes / 16;  // vectors per row
    uint4* base = reinterpret_cast<uint4*>(static_cast<uint8_t*>(kv ? a.vc : a.kc) +
                                           ((long long)layer * a.layer_stride + (long long)slot * a.slot_stride +
                                            ((long long)h * a.cap + n_ctx) * a.hd) * a.elem_bytes);
    const int total = n * vpr, rows_step = 32 / vpr, rest = 32 - rows_step * vpr;
    int i = lane / vpr, c = lane - i * vpr;  // row and vector of this lane's next one
    for (int v0 = 0; v0 < total; v0 += 32 * KC_VEC) {
        uint4 r[KC_VEC];
        unsigned moved = 0;
#pragma unroll
        for (int u = 0; u < KC_VEC; ++u) {
            if (v0 + u * 32 + lane < total) {
                const int p = path[i];
                if (p != i) {
                    r[u] = base[(long long)p * vpr + c];
                    moved |= 1u << u;
                }
            }
            i += rows_step;
            c += rest;
            if (c >= vpr) {
                c -= vpr;
                ++i;
            }
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < KC_VEC; ++u)
            if (moved >> u & 1) base[v0 + u * 32 + lane] = r[u];
        __syncwarp();
    }
}

// ---- the drafted nodes' rows: RoPE of q (in place) and k at the node's depth, K / V store -------------
// Node m of the sequence in slots[m] stands at position pos[slot] + depth[m] and takes cache row
// pos[slot] + m (siblings share a position).  One CTA per (node, head), a thread per rotation pair,
// as the prefill chunk's kernel.  (A launch's latency: q, k and v of a step's 64 nodes are 1 to 2 MB,
// which the attention behind it reads from L2.)
__global__ void tf_tree_rope_store_kernel(const AttnArgs a, const int* depth) {
    pdl_trigger();
    pdl_wait();
    const int m = blockIdx.x, h = blockIdx.y, j = threadIdx.x;
    const int hd = a.hd, d2 = hd / 2;
    const int slot = a.slots[m], row_pos = a.pos[slot] + m, pos = a.pos[slot] + depth[m];
    if (a.pos[slot] < 0 || row_pos >= a.cap || depth[m] < 0 || depth[m] > m) {
        if (j == 0) atomicCAS(a.err, 0, ERR_POS);
        return;
    }
    float* row = const_cast<float*>(a.qkv) + (size_t)m * a.ld_qkv;
    const float c = a.cosb[(size_t)pos * d2 + j], sn = a.sinb[(size_t)pos * d2 + j];
    if (h < a.n_head) {
        float* q = row + (size_t)h * hd;
        float x0 = q[j], x1 = q[j + d2];
        rope_pair(x0, x1, c, sn);
        q[j] = x0;
        q[j + d2] = x1;
    } else {
        const int kvh = h - a.n_head;
        const float* k = row + (size_t)a.n_head * hd + (size_t)kvh * hd;
        const float* v = row + (size_t)(a.n_head + a.n_kv) * hd + (size_t)kvh * hd;
        float x0 = k[j], x1 = k[j + d2];
        rope_pair(x0, x1, c, sn);
        const size_t off = (size_t)slot * a.slot_stride + (size_t)kvh * a.cap * hd + (size_t)row_pos * hd;
        kv_store(a.kc, (long long)(off + j), a.kv_type, x0);
        kv_store(a.kc, (long long)(off + j + d2), a.kv_type, x1);
        kv_store(a.vc, (long long)(off + j), a.kv_type, v[j]);
        kv_store(a.vc, (long long)(off + j + d2), a.kv_type, v[j + d2]);
    }
}

cudaError_t tree_rope_store_launch(const AttnArgs& a, const int* depth, int M, cudaStream_t st) {
    if (a.hd > AT_MAX_HD || a.hd % 2) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(M, a.n_head + a.n_kv);
    cfg.blockDim = dim3(a.hd / 2);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, tf_tree_rope_store_kernel, a, depth);
}

cudaError_t kv_commit_launch(const KvCommitArgs& a, cudaStream_t st) {
    const long long warps = (long long)a.n_layer * a.B * a.n_kv * 2, per = KC_THREADS / 32;
    if (warps > 0xFFFFFFFFll - KC_THREADS) return cudaErrorInvalidValue;
    tf_kv_commit_kernel<<<(unsigned)((warps + per - 1) / per), KC_THREADS, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace tfb
