// Op-level C-ABI of the quantised KV cache: argument checks, then the launchers of kvq.cuh.
#include <string>

#include "engine.cuh"
#include "kvq.cuh"

using namespace tfb;

namespace {
int kvq_status(cudaError_t e, const char* what) {
    if (e != cudaSuccess) return set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return 0;
}
bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// A row operand [rows][ld] of `width` floats (nullptr: absent)
int row_operand(const void* p, int ld, int width) {
    if (!p) return 0;
    if (!aligned(p, 16)) return set_error("rows must be 16-byte aligned");
    if (ld < width || ld % 4) return set_error("a row stride must be a multiple of 4, at least heads * head_dim");
    return 0;
}
int cache_shape(const void* kc, const void* vc, int kv_type, long long slot_stride, int cap, int n_slots, int n_kv_heads,
                int head_dim) {
    if (kv_type != KV_Q4_0 && kv_type != KV_Q8_0) return set_error("kv_type must be TF_KV_Q4_0 or TF_KV_Q8_0");
    if (n_kv_heads < 1 || n_kv_heads > 1024) return set_error("n_kv_heads must be in [1, 1024]");
    if (head_dim <= 0 || head_dim % 32 || head_dim > KVQ_MAX_HD)
        return set_error("head_dim must be a positive multiple of 32 up to 128");
    if (cap < 16 || cap % 16 || cap > 1 << 30) return set_error("cap must be a positive multiple of 16, at most 2^30");
    if (n_slots < 1 || slot_stride < (long long)n_kv_heads * cap * head_dim || slot_stride % (16 * head_dim))
        return set_error("slot_stride must be a multiple of 16 * head_dim, at least n_kv_heads * cap * head_dim");
    if (!kc || !vc) return set_error("null pointer");
    if (!aligned(kc, 16) || !aligned(vc, 16)) return set_error("the caches must be 16-byte aligned");
    return 0;
}
long long cache_bytes(int kv_type, long long elements) { return elements / 32 * (kv_type == KV_Q4_0 ? 18 : 34); }

int rope_shape(const float* freq, int rope_dim, int head_dim, const int* pos) {
    if (!freq) return 0;
    if (rope_dim <= 0 || rope_dim % 8 || rope_dim > head_dim)
        return set_error("rope_dim must be a positive multiple of 8, at most head_dim");
    if (!pos) return set_error("pos must not be null with a rotation");
    return 0;
}
int weights_ok(const float* wq, const float* wk, float eps) {
    if (!aligned(wq, 16) || !aligned(wk, 16)) return set_error("norm weights must be 16-byte aligned");
    if ((wq || wk) && !(eps >= 0.0f)) return set_error("eps must not be negative or NaN");
    return 0;
}
template <class A>
void set_cache(A& a, int kv_type, long long slot_stride, int cap, int n_slots, int n_kv_heads, int head_dim) {
    a.bits = kvq_bits(kv_type);
    a.slot_bytes = cache_bytes(kv_type, slot_stride);
    a.head_bytes = cache_bytes(kv_type, (long long)cap * head_dim);
    a.cap = cap;
    a.n_slots = n_slots;
    a.n_kv = n_kv_heads;
    a.hd = head_dim;
}

int attn_shape(int B, int T, int n_heads, int n_kv_heads, int head_dim) {
    if (B < 0 || B > 65535) return set_error("B must be in [0, 65535]");
    if (T < 1 || T > KVQ_MAX_ROWS) return set_error("T must be in [1, 64]");
    if (n_heads <= 0 || n_heads > 1024 || n_kv_heads <= 0 || n_heads % n_kv_heads)
        return set_error("n_heads must be a positive multiple of n_kv_heads, at most 1024");
    if (head_dim <= 0 || head_dim % 32 || head_dim > KVQ_MAX_HD)
        return set_error("head_dim must be a positive multiple of 32 up to 128");
    return 0;
}
}  // namespace

extern "C" {

int tf_op_qk_norm_rope(float* q_out, int ld_qo, float* k_out, int ld_ko, const float* q, int ld_q, const float* k, int ld_k,
                       const float* q_weight, const float* k_weight, float eps, const float* freq, int rope_dim,
                       const int* pos, int rows, int n_heads, int n_kv_heads, int head_dim, void* stream) {
    if (rows < 0) return set_error("rows must not be negative");
    if (!q && !k) return set_error("q and k are both null");
    if ((q != nullptr) != (q_out != nullptr) || (k != nullptr) != (k_out != nullptr))
        return set_error("q and q_out, k and k_out come together");
    if ((q && (n_heads < 1 || n_heads > 1024)) || (k && (n_kv_heads < 1 || n_kv_heads > 1024)))
        return set_error("heads must be in [1, 1024]");
    if (head_dim <= 0 || head_dim % 8 || head_dim > KVQ_MAX_HD)
        return set_error("head_dim must be a positive multiple of 8 up to 128");
    if (rope_shape(freq, rope_dim, head_dim, pos) || weights_ok(q_weight, k_weight, eps)) return -1;
    if (row_operand(q, ld_q, n_heads * head_dim) || row_operand(q_out, ld_qo, n_heads * head_dim) ||
        row_operand(k, ld_k, n_kv_heads * head_dim) || row_operand(k_out, ld_ko, n_kv_heads * head_dim))
        return -1;
    if (rows == 0) return 0;
    KvqRowsArgs a = {};
    a.q = q;
    a.ld_q = ld_q;
    a.q_out = q_out;
    a.ld_qo = ld_qo;
    a.k = k;
    a.ld_k = ld_k;
    a.k_out = k_out;
    a.ld_ko = ld_ko;
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.eps = eps;
    a.freq = freq;
    a.rot = freq ? rope_dim : 0;
    a.pos = pos;
    a.bits = 4;
    a.rows = rows;
    a.n_head = n_heads;
    a.n_kv = n_kv_heads;
    a.hd = head_dim;
    return kvq_status(kvq_rows_launch(a, static_cast<cudaStream_t>(stream)), "qk_norm_rope");
}

int tf_op_kv_quant(void* k_cache, void* v_cache, int kv_type, long long slot_stride, int cap, int n_slots, const int* slots,
                   const int* pos, const float* k, int ld_k, const float* v, int ld_v, int rows, int n_kv_heads, int head_dim,
                   void* stream) {
    if (rows < 0) return set_error("rows must not be negative");
    if (cache_shape(k_cache, v_cache, kv_type, slot_stride, cap, n_slots, n_kv_heads, head_dim)) return -1;
    if (!pos || !k || !v) return set_error("null pointer");
    if (row_operand(k, ld_k, n_kv_heads * head_dim) || row_operand(v, ld_v, n_kv_heads * head_dim)) return -1;
    if (rows == 0) return 0;
    KvqRowsArgs a = {};
    if (op_err_word(&a.err)) return -1;
    set_cache(a, kv_type, slot_stride, cap, n_slots, n_kv_heads, head_dim);
    a.kc = static_cast<uint8_t*>(k_cache);
    a.vc = static_cast<uint8_t*>(v_cache);
    a.k = k;
    a.ld_k = ld_k;
    a.v = v;
    a.ld_v = ld_v;
    a.slots = slots;
    a.pos = pos;
    a.rows = rows;
    return kvq_status(kvq_rows_launch(a, static_cast<cudaStream_t>(stream)), "kv_quant");
}

int tf_op_kv_dequant(float* k, int ld_k, float* v, int ld_v, const void* k_cache, const void* v_cache, int kv_type,
                     long long slot_stride, int cap, int n_slots, const int* slots, const int* pos, int rows, int n_kv_heads,
                     int head_dim, void* stream) {
    if (rows < 0) return set_error("rows must not be negative");
    if (cache_shape(k_cache, v_cache, kv_type, slot_stride, cap, n_slots, n_kv_heads, head_dim)) return -1;
    if (!pos || (!k && !v)) return set_error("null pointer");
    if (row_operand(k, ld_k, n_kv_heads * head_dim) || row_operand(v, ld_v, n_kv_heads * head_dim)) return -1;
    if (rows == 0) return 0;
    KvqReadArgs a = {};
    if (op_err_word(&a.err)) return -1;
    set_cache(a, kv_type, slot_stride, cap, n_slots, n_kv_heads, head_dim);
    a.kc = static_cast<const uint8_t*>(k_cache);
    a.vc = static_cast<const uint8_t*>(v_cache);
    a.k = k;
    a.ld_k = ld_k;
    a.v = v;
    a.ld_v = ld_v;
    a.slots = slots;
    a.pos = pos;
    a.rows = rows;
    return kvq_status(kvq_read_launch(a, static_cast<cudaStream_t>(stream)), "kv_dequant");
}

int tf_op_qkv_store(float* q_out, int ld_qo, void* k_cache, void* v_cache, int kv_type, long long slot_stride, int cap,
                    int n_slots, const int* slots, const int* pos, const float* q, int ld_q, const float* k, int ld_k,
                    const float* v, int ld_v, const float* q_weight, const float* k_weight, float eps, const float* freq,
                    int rope_dim, int rows, int n_heads, int n_kv_heads, int head_dim, void* stream) {
    if (rows < 0) return set_error("rows must not be negative");
    if (cache_shape(k_cache, v_cache, kv_type, slot_stride, cap, n_slots, n_kv_heads, head_dim)) return -1;
    if (n_heads < 1 || n_heads > 1024) return set_error("heads must be in [1, 1024]");
    if (!pos || !q || !q_out || !k || !v) return set_error("null pointer");
    if (rope_shape(freq, rope_dim, head_dim, pos) || weights_ok(q_weight, k_weight, eps)) return -1;
    if (row_operand(q, ld_q, n_heads * head_dim) || row_operand(q_out, ld_qo, n_heads * head_dim) ||
        row_operand(k, ld_k, n_kv_heads * head_dim) || row_operand(v, ld_v, n_kv_heads * head_dim))
        return -1;
    if (rows == 0) return 0;
    KvqRowsArgs a = {};
    if (op_err_word(&a.err)) return -1;
    set_cache(a, kv_type, slot_stride, cap, n_slots, n_kv_heads, head_dim);
    a.kc = static_cast<uint8_t*>(k_cache);
    a.vc = static_cast<uint8_t*>(v_cache);
    a.q = q;
    a.ld_q = ld_q;
    a.q_out = q_out;
    a.ld_qo = ld_qo;
    a.k = k;
    a.ld_k = ld_k;
    a.v = v;
    a.ld_v = ld_v;
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.eps = eps;
    a.freq = freq;
    a.rot = freq ? rope_dim : 0;
    a.slots = slots;
    a.pos = pos;
    a.rows = rows;
    a.n_head = n_heads;
    return kvq_status(kvq_rows_launch(a, static_cast<cudaStream_t>(stream)), "qkv_store");
}

int tf_op_attn_quant_workspace(int B, int T, int n_heads, int n_kv_heads, int head_dim, size_t* bytes) {
    if (!bytes) return set_error("bytes is null");
    *bytes = 0;
    if (attn_shape(B, T, n_heads, n_kv_heads, head_dim)) return -1;
    *bytes = kvq_attn_ws_bytes(T, n_heads, n_kv_heads, head_dim);
    return 0;
}

int tf_op_attn_quant(float* out, int ld_out, const float* q, int ld_q, const void* k_cache, const void* v_cache, int kv_type,
                     long long slot_stride, int cap, int n_slots, const int* slots, const int* n_ctx, const int* n_new, int B,
                     int T, int n_heads, int n_kv_heads, int head_dim, void* ws, size_t ws_bytes, void* stream) {
    if (attn_shape(B, T, n_heads, n_kv_heads, head_dim)) return -1;
    if (cache_shape(k_cache, v_cache, kv_type, slot_stride, cap, n_slots, n_kv_heads, head_dim)) return -1;
    if (!out || !q || !n_ctx || !ws) return set_error("null pointer");
    if (row_operand(out, ld_out, n_heads * head_dim) || row_operand(q, ld_q, n_heads * head_dim)) return -1;
    if (!aligned(ws, 256)) return set_error("the workspace must be 256-byte aligned");
    if (ws_bytes < kvq_attn_ws_bytes(T, n_heads, n_kv_heads, head_dim)) return set_error("workspace too small");
    if (!kvq_attn_fits(B, T, n_heads, n_kv_heads, cap))
        return set_error("B * n_kv_heads * ceil(T * (n_heads / n_kv_heads) / 4) * (cap / 16 + 24) must be below 2^31");
    if (B == 0) return 0;
    KvqAttnArgs a = {};
    if (op_err_word(&a.err)) return -1;
    set_cache(a, kv_type, slot_stride, cap, n_slots, n_kv_heads, head_dim);
    a.out = out;
    a.ld_out = ld_out;
    a.q = q;
    a.ld_q = ld_q;
    a.kc = static_cast<const uint8_t*>(k_cache);
    a.vc = static_cast<const uint8_t*>(v_cache);
    a.slots = slots;
    a.n_ctx = n_ctx;
    a.n_new = n_new;
    a.B = B;
    a.T = T;
    a.n_head = n_heads;
    a.ws = ws;
    return kvq_status(kvq_attn_launch(a, static_cast<cudaStream_t>(stream)), "attn_quant");
}

}  // extern "C"
