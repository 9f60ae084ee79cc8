// A KV cache in Q4_0 / Q8_0: its layout, arguments and launchers of the row operators (kvq_rows.cu: norms
// with the rotation, writing, reading back) and of the attention over it (kvq_attn.cu).
//
// Layout: [slot][kv head][cap / 16][block], a block being 16 positions: the codes (16 hd bits / 8 bytes), then
// the scales (f16, one per position and group of 32 dims), together what 16 hd / 32 GGUF blocks take.  Codes
// lie as mma.m16n8k16 wants its A operand, 32-bit word by word: word i of lane l belongs to the fragment that
// lane l feeds, and lanes' words are gathered in vectors of four (the last two of an odd number of pairs in
// vectors of two), so that a warp reads a block in 16-byte loads that follow one another.
//   K, position p, dim e:  lane = 4 (p % 8) + e % 32 / 8
//      Q4_0: word = (p / 8) (hd / 32) + e / 32, nibble e % 8;  Q8_0: word = 2 (that) + e % 8 / 4, byte e % 4
//   V, position p, dim e:  lane = 4 (e % 16 / 2) + p % 8 / 2, byte 2 (p % 2) + p / 8
//      Q4_0: word = e / 16, nibble e % 2 of the byte;  Q8_0: word = 2 (e / 16) + e % 2
//   scale of position p, group k: index (2 (p % 8) + p / 8) hd / 32 + k
// A byte holds codes of one position, so that rows are written without reading their neighbours.
// Value = (code - 8) scale, or (code - 128) scale.
#pragma once

#include "common.cuh"

namespace tfb {

enum : int { KV_Q4_0 = 3, KV_Q8_0 = 4 };
constexpr int KVQ_MAX_HD = 128;
constexpr int KVQ_MAX_ROWS = 64;  // new rows per sequence of the attention

__host__ __device__ constexpr int kvq_bits(int kv_type) { return kv_type == KV_Q4_0 ? 4 : 8; }
__host__ __device__ constexpr int kvq_code_bytes(int bits, int hd) { return 2 * hd * bits; }
__host__ __device__ constexpr int kvq_block_bytes(int bits, int hd) { return 2 * hd * bits + hd; }

// Byte of word i of a lane within a block whose lanes have `words` words each.
__host__ __device__ __forceinline__ int kvq_word(int words, int i, int lane) {
    const int whole = words & ~3;
    return (i < whole ? (i >> 2) * 512 + lane * 16 : (whole >> 2) * 512 + lane * 8) + (i & 3) * 4;
}

// ---- rows: norm, rotation, writing, reading (kvq_rows.cu) --------------------------------------------
struct KvqRowsArgs {
    const float* q;         // [rows][ld_q]: n_head * hd (nullptr: no queries)
    int ld_q;
    float* q_out;
    int ld_qo;
    const float* k;         // [rows][ld_k]: n_kv * hd (nullptr: no keys)
    int ld_k;
    float* k_out;           // nullptr: keys go to the cache only
    int ld_ko;
    const float* v;         // [rows][ld_v] (nullptr: no values)
    int ld_v;
    const float* q_weight;  // [hd] (nullptr: no norm)
    const float* k_weight;
    float eps;
    const float* freq;      // [rot / 2] (nullptr: no rotation)
    int rot;
    uint8_t* kc;            // nullptr: no cache
    uint8_t* vc;
    int bits;
    long long slot_bytes, head_bytes;
    int cap, n_slots;
    const int* slots;       // [rows] (nullptr: row r in slot r); below 0: the row is left out
    const int* pos;         // [rows]
    int rows, n_head, n_kv, hd;
    int* err;
};
cudaError_t kvq_rows_launch(const KvqRowsArgs& a, cudaStream_t st);

struct KvqReadArgs {
    float* k;               // [rows][ld_k] (nullptr: values only)
    int ld_k;
    float* v;
    int ld_v;
    const uint8_t* kc;
    const uint8_t* vc;
    int bits;
    long long slot_bytes, head_bytes;
    int cap, n_slots;
    const int* slots;
    const int* pos;
    int rows, n_kv, hd;
    int* err;
};
cudaError_t kvq_read_launch(const KvqReadArgs& a, cudaStream_t st);

// ---- attention (kvq_attn.cu) --------------------------------------------------------------------------
struct KvqAttnArgs {
    float* out;             // [B*T][ld_out]: n_head * hd per row
    int ld_out;
    const float* q;         // [B*T][ld_q]
    int ld_q;
    const uint8_t* kc;
    const uint8_t* vc;
    int bits;
    long long slot_bytes, head_bytes;
    int cap, n_slots;
    const int* slots;       // [B] (nullptr: b)
    const int* n_ctx;       // [B]: positions before the new rows
    const int* n_new;       // [B] (nullptr: T)
    int B, T, n_head, n_kv, hd;
    void* ws;
    int* err;
};
size_t kvq_attn_ws_bytes(int T, int n_head, int n_kv, int hd);     // any B
bool kvq_attn_fits(int B, int T, int n_head, int n_kv, int cap);   // blocks are counted in 32 bits
cudaError_t kvq_attn_launch(const KvqAttnArgs& a, cudaStream_t st);

}  // namespace tfb
