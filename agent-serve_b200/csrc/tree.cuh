// Speculative decoding with a tree of drafted tokens: arguments and launchers of the tree
// attention (tree_attn.cu), the verification walk (tree_verify.cu) and the cache commit
// (tree_commit.cu).
#pragma once

#include "attention.cuh"

namespace tfb {

constexpr int TREE_MAX_NODES = 256;  // drafted tokens per sequence, the root included

// Attention of B trees of up to T nodes over one layer's cache.  Sequence b holds n_ctx[b]
// committed positions in cache slot slots[b]; its nodes' keys and values are the next
// n_node[b] rows.  Node t sees every committed position and node j where bit j of
// mask[b][t][] is set (nullptr: j <= t, a chain).
struct TreeAttnArgs {
    float* out;             // [B*T][ld_out]: n_head * hd per row
    int ld_out;
    const float* q;         // [B*T][ld_q]
    int ld_q;
    const void* kc;         // [n_slots][n_kv][cap][hd], slots slot_stride elements apart
    const void* vc;
    int kv_type;
    long long slot_stride;
    int cap, n_slots;
    const int* slots;       // [B] (nullptr: b)
    const int* n_ctx;       // [B]
    const int* n_node;      // [B] (nullptr: T)
    const unsigned long long* mask;  // [B][T][ceil(T / 64)]
    int B, T, n_head, n_kv, hd;
    void* ws;
    int* err;
};
size_t tree_attn_ws_bytes(int T, int n_head, int n_kv, int hd);  // any B
bool tree_attn_fits(int B, int T, int n_head, int n_kv, int cap);  // tiles are counted in 32 bits
cudaError_t tree_attn_launch(const TreeAttnArgs& a, cudaStream_t st, bool pdl);

struct TreeVerifyArgs {
    int* path;              // [B][T]: accepted nodes, the root first, -1 behind them
    int* n_path;            // [B]
    int* next;              // [B]: the token after the path
    const float* logits;    // [B*T][ld]
    long long ld;
    const float* draft;     // [B*T][ld_draft] or nullptr
    long long ld_draft;
    const int* tokens;      // [B][T]
    const int* parents;     // [B][T]
    const int* n_node;      // [B] (nullptr: T)
    const float* u;         // [B][T]
    float inv_temp;         // 0: greedy
    int B, T, V;
    void* ws;
    int* err;
};
size_t tree_verify_ws_bytes(int B, int T, int V);
int tree_verify_max_vocab(bool draft);  // a row's slices fit the shared memory of a cluster
// What a caller's temperature and vocabulary are refused for (nullptr: nothing); inv_temp: 0 for greedy.
const char* tree_verify_refusal(float temperature, bool draft, int V, float* inv_temp);
cudaError_t tree_verify_launch(const TreeVerifyArgs& a, cudaStream_t st);

struct KvCommitArgs {
    void* kc;               // [n_layer][n_slots][n_kv][cap][hd]
    void* vc;
    int elem_bytes;
    int n_layer;
    long long layer_stride, slot_stride;  // elements
    int cap, n_slots;
    const int* slots;       // [B] (nullptr: b)
    const int* n_ctx;       // [B]
    const int* path;        // [B][ld_path]
    int ld_path;
    const int* n_path;      // [B]
    int* n_new;             // [B] or nullptr
    int B, n_kv, hd;
    int* err;
};
cudaError_t kv_commit_launch(const KvCommitArgs& a, cudaStream_t st);
// RoPE at each node's depth and K / V store of a tree step's M nodes (AttnArgs of the step)
cudaError_t tree_rope_store_launch(const AttnArgs& a, const int* depth, int M, cudaStream_t st);

}  // namespace tfb
