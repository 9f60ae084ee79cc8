// Op-level C-ABI of speculative decoding: argument checks, then the launchers of tree.cuh.
#include <cmath>
#include <string>

#include "engine.cuh"
#include "tree.cuh"

using namespace tfb;

namespace {
int tree_status(cudaError_t e, const char* what) {
    if (e != cudaSuccess) return set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return 0;
}
bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool kv_ok(int t) { return t == KV_F32 || t == KV_F16 || t == KV_BF16; }

int attn_shape(int B, int T, int n_heads, int n_kv_heads, int head_dim) {
    if (B < 0 || B > 65535) return set_error("B must be in [0, 65535]");
    if (T < 1 || T > TREE_MAX_NODES) return set_error("T must be in [1, 256]");
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads)
        return set_error("n_heads must be a positive multiple of n_kv_heads");
    if (n_heads > 1024 || n_heads / n_kv_heads > AT_MAX_REP)
        return set_error("at most 1024 heads and 8 query heads per kv head");
    if (head_dim <= 0 || head_dim % 8 || head_dim > AT_MAX_HD)
        return set_error("head_dim must be a positive multiple of 8 up to 128");
    return 0;
}
int verify_shape(int B, int T, int V) {
    if (B < 0 || B > 65535) return set_error("B must be in [0, 65535]");
    if (T < 1 || T > TREE_MAX_NODES) return set_error("T must be in [1, 256]");
    if (V < 1) return set_error("V must be positive");
    return 0;
}
}  // namespace

namespace tfb {
const char* tree_verify_refusal(float temperature, bool draft, int V, float* inv_temp) {
    if (temperature != temperature) return "temperature is NaN";
    *inv_temp = temperature <= 0.0f ? 0.0f : (float)(1.0 / (double)temperature);
    if (!(*inv_temp < INFINITY) || (temperature > 0.0f && *inv_temp == 0.0f)) return "temperature out of range";
    if (V > tree_verify_max_vocab(draft && temperature > 0.0f)) return "V is above the limit (409600 with draft, 819200 without)";
    return nullptr;
}
}  // namespace tfb

extern "C" {

int tf_tree_mask(const int* parents, int n, int T, unsigned long long* mask, int* depth) {
    if (!parents || !mask) return set_error("null parents or mask");
    if (T < 1 || T > TREE_MAX_NODES || n < 0 || n > T) return set_error("T must be in [1, 256] and n in [0, T]");
    for (int t = 0; t < n; ++t)
        if (t == 0 ? parents[0] >= 0 : (parents[t] < 0 || parents[t] >= t))
            return set_error("node 0 is the root (parent < 0), every other node's parent precedes it");
    const int W = (T + 63) / 64;
    for (int t = 0; t < T; ++t)
        for (int w = 0; w < W; ++w) {
            unsigned long long m = t < n && t > 0 ? mask[(size_t)parents[t] * W + w] : 0ull;
            if (t < n && w == t / 64) m |= 1ull << (t % 64);
            mask[(size_t)t * W + w] = m;
        }
    if (depth)
        for (int t = 0; t < T; ++t) depth[t] = t < n && t > 0 ? depth[parents[t]] + 1 : 0;
    return 0;
}

int tf_op_attn_tree_workspace(int B, int T, int n_heads, int n_kv_heads, int head_dim, size_t* bytes) {
    if (!bytes) return set_error("bytes is null");
    *bytes = 0;
    if (attn_shape(B, T, n_heads, n_kv_heads, head_dim)) return -1;
    *bytes = tree_attn_ws_bytes(T, n_heads, n_kv_heads, head_dim);
    return 0;
}

int tf_op_attn_tree(float* out, int ld_out, const float* q, int ld_q, const void* k_cache, const void* v_cache, int kv_type,
                    long long slot_stride, int cap, int n_slots, const int* slots, const int* n_ctx, const int* n_node,
                    const unsigned long long* mask, int B, int T, int n_heads, int n_kv_heads, int head_dim, void* ws,
                    size_t ws_bytes, void* stream) {
    if (attn_shape(B, T, n_heads, n_kv_heads, head_dim)) return -1;
    if (B == 0) return 0;
    if (!out || !q || !k_cache || !v_cache || !n_ctx || !ws) return set_error("null pointer");
    if (!kv_ok(kv_type)) return set_error("unknown kv_type");
    if (ld_out < n_heads * head_dim || ld_q < n_heads * head_dim || ld_out % 4 || ld_q % 4)
        return set_error("ld_out and ld_q must be multiples of 4, at least n_heads * head_dim");
    if (cap < 1 || cap > 1 << 30 || n_slots < 1 || slot_stride < (long long)n_kv_heads * cap * head_dim || slot_stride % 8)
        return set_error("bad cache shape (cap, n_slots, slot_stride)");
    if (!aligned(out, 16) || !aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(ws, 256))
        return set_error("out, q and the caches must be 16-byte aligned, the workspace 256-byte aligned");
    if (ws_bytes < tree_attn_ws_bytes(T, n_heads, n_kv_heads, head_dim)) return set_error("workspace too small");
    if (!tree_attn_fits(B, T, n_heads, n_kv_heads, cap))
        return set_error("B * n_kv_heads * ceil(T * (n_heads / n_kv_heads) / 16) * (cap / 32 + 8) must be below 2^31");
    TreeAttnArgs a = {};
    if (op_err_word(&a.err)) return -1;
    a.out = out;
    a.ld_out = ld_out;
    a.q = q;
    a.ld_q = ld_q;
    a.kc = k_cache;
    a.vc = v_cache;
    a.kv_type = kv_type;
    a.slot_stride = slot_stride;
    a.cap = cap;
    a.n_slots = n_slots;
    a.slots = slots;
    a.n_ctx = n_ctx;
    a.n_node = n_node;
    a.mask = mask;
    a.B = B;
    a.T = T;
    a.n_head = n_heads;
    a.n_kv = n_kv_heads;
    a.hd = head_dim;
    a.ws = ws;
    return tree_status(tree_attn_launch(a, static_cast<cudaStream_t>(stream), false), "attn_tree");
}

int tf_op_verify_tree_workspace(int B, int T, int V, size_t* bytes) {
    if (!bytes) return set_error("bytes is null");
    *bytes = 0;
    if (verify_shape(B, T, V)) return -1;
    *bytes = tree_verify_ws_bytes(B, T, V);
    return 0;
}

int tf_op_verify_tree(int* path, int* n_path, int* next, const float* logits, long long ld, const float* draft,
                      long long ld_draft, const int* tokens, const int* parents, const int* n_node, const float* u,
                      float temperature, int B, int T, int V, void* ws, size_t ws_bytes, void* stream) {
    if (verify_shape(B, T, V)) return -1;
    if (B == 0) return 0;
    if (!path || !n_path || !next || !logits || !tokens || !parents || !ws) return set_error("null pointer");
    if (!(temperature <= 0.0f) && !u) return set_error("u must not be null at a positive temperature");
    float inv = 0.0f;
    const char* refusal = tree_verify_refusal(temperature, draft != nullptr, V, &inv);
    if (refusal) return set_error(refusal);
    if (ld < V || (draft && ld_draft < V)) return set_error("ld must be at least V");
    if (!aligned(ws, 256)) return set_error("the workspace must be 256-byte aligned");
    if (ws_bytes < tree_verify_ws_bytes(B, T, V)) return set_error("workspace too small");
    TreeVerifyArgs a = {};
    if (op_err_word(&a.err)) return -1;
    a.path = path;
    a.n_path = n_path;
    a.next = next;
    a.logits = logits;
    a.ld = ld;
    a.draft = temperature <= 0.0f ? nullptr : draft;
    a.ld_draft = ld_draft;
    a.tokens = tokens;
    a.parents = parents;
    a.n_node = n_node;
    a.u = u;
    a.inv_temp = inv;
    a.B = B;
    a.T = T;
    a.V = V;
    a.ws = ws;
    return tree_status(tree_verify_launch(a, static_cast<cudaStream_t>(stream)), "verify_tree");
}

int tf_op_kv_commit(void* k_cache, void* v_cache, int kv_type, int n_layer, long long layer_stride, long long slot_stride,
                    int cap, int n_slots, const int* slots, const int* n_ctx, const int* path, int ld_path,
                    const int* n_path, int* n_new, int B, int n_kv_heads, int head_dim, void* stream) {
    if (B < 0 || B > 65535) return set_error("B must be in [0, 65535]");
    if (n_layer < 1 || n_kv_heads < 1 || cap < 1 || n_slots < 1 || ld_path < 1) return set_error("bad cache or path shape");
    if (head_dim <= 0 || head_dim % 8) return set_error("head_dim must be a positive multiple of 8");
    if (!kv_ok(kv_type)) return set_error("unknown kv_type");
    if (slot_stride < (long long)n_kv_heads * cap * head_dim || slot_stride % 8 || layer_stride % 8 ||
        (n_layer > 1 && layer_stride < slot_stride))
        return set_error("bad cache strides");
    if (B == 0) return 0;
    if (!k_cache || !v_cache || !n_ctx || !path || !n_path) return set_error("null pointer");
    auto in_n_new = [&](const int* p, long long n) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(n_new), y = reinterpret_cast<uintptr_t>(p);
        return n_new && p && x < y + sizeof(int) * n && y < x + sizeof(int) * B;
    };
    if (in_n_new(n_ctx, B) || in_n_new(n_path, B) || in_n_new(slots, B) || in_n_new(path, (long long)B * ld_path))
        return set_error("n_new must not overlap n_ctx, n_path, slots or path (every block of the launch reads them)");
    if (!aligned(k_cache, 16) || !aligned(v_cache, 16)) return set_error("the caches must be 16-byte aligned");
    KvCommitArgs a = {};
    if (op_err_word(&a.err)) return -1;
    a.kc = k_cache;
    a.vc = v_cache;
    a.elem_bytes = kv_type == KV_F32 ? 4 : 2;
    a.n_layer = n_layer;
    a.layer_stride = layer_stride;
    a.slot_stride = slot_stride;
    a.cap = cap;
    a.n_slots = n_slots;
    a.slots = slots;
    a.n_ctx = n_ctx;
    a.path = path;
    a.ld_path = ld_path;
    a.n_path = n_path;
    a.n_new = n_new;
    a.B = B;
    a.n_kv = n_kv_heads;
    a.hd = head_dim;
    return tree_status(kv_commit_launch(a, static_cast<cudaStream_t>(stream)), "kv_commit");
}

}  // extern "C"
