// Commit of an accepted path of drafted nodes: cache row n_ctx + i <- row n_ctx + path[i], in
// place, for K and V of every layer and kv head, so that the path's rows follow the committed
// context without gaps.
//
// One warp per (layer, sequence, kv head, K or V).  The path is strictly increasing, so
// path[i] >= i: taking the rows in ascending groups, each group loaded into registers before it
// is stored, never reads a row that an earlier group has overwritten.  Bound by latency (a few
// rows of 128 to 512 bytes per warp); rows that stay where they are (the root's) are not moved.
#include "tree.cuh"

namespace tfb {

constexpr int KC_THREADS = 128;
constexpr int KC_VEC = 8;  // 16-byte vectors in flight per lane

__global__ void __launch_bounds__(KC_THREADS) tf_kv_commit_kernel(const KvCommitArgs a) {
    const int lane = threadIdx.x & 31;
    const long long unit = ((long long)blockIdx.x * KC_THREADS + threadIdx.x) >> 5;  // layer, sequence, kv head, K / V
    if (unit >= (long long)a.n_layer * a.B * a.n_kv * 2) return;
    const int kv = (int)(unit & 1);
    const int h = (int)((unit >> 1) % a.n_kv);
    const int b = (int)((unit >> 1) / a.n_kv % a.B);
    const int layer = (int)((unit >> 1) / a.n_kv / a.B);
    const int slot = a.slots ? a.slots[b] : b, n_ctx = a.n_ctx[b], n = a.n_path[b];
    const int* path = a.path + (long long)b * a.ld_path;
    bool bad = slot < 0 || slot >= a.n_slots || n_ctx < 0 || n_ctx > a.cap || n < 0 || n > a.ld_path;
    if (!bad)
        for (int i = lane; i < n; i += 32) {
            const int p = path[i];
            bad |= p < i || p >= a.cap - n_ctx || (i > 0 && p <= path[i - 1]);
        }
    bad = __any_sync(0xFFFFFFFFu, bad);
    if (unit < 2ll * a.n_kv * a.B && kv == 0 && h == 0 && lane == 0) {
        if (bad) atomicCAS(a.err, 0, ERR_POS);
        if (a.n_new) a.n_new[b] = bad ? n_ctx : n_ctx + n;
    }
    if (bad || n == 0) return;
    const int vpr = a.hd * a.elem_bytes / 16;  // vectors per row
    uint4* base = reinterpret_cast<uint4*>(static_cast<uint8_t*>(kv ? a.vc : a.kc) +
                                           ((long long)layer * a.layer_stride + (long long)slot * a.slot_stride +
                                            ((long long)h * a.cap + n_ctx) * a.hd) * a.elem_bytes);
    const int total = n * vpr;
    for (int v0 = 0; v0 < total; v0 += 32 * KC_VEC) {
        uint4 r[KC_VEC];
#pragma unroll
        for (int u = 0; u < KC_VEC; ++u) {
            const int v = v0 + u * 32 + lane;
            if (v < total) {
                const int i = v / vpr, p = path[i];
                if (p != i) r[u] = base[(long long)p * vpr + v % vpr];
            }
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < KC_VEC; ++u) {
            const int v = v0 + u * 32 + lane;
            if (v < total) {
                const int i = v / vpr;
                if (path[i] != i) base[v] = r[u];
            }
        }
        __syncwarp();
    }
}

cudaError_t kv_commit_launch(const KvCommitArgs& a, cudaStream_t st) {
    const long long warps = (long long)a.n_layer * a.B * a.n_kv * 2, per = KC_THREADS / 32;
    if ((warps + per - 1) / per > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    tf_kv_commit_kernel<<<(unsigned)((warps + per - 1) / per), KC_THREADS, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace tfb
