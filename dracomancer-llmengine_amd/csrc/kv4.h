// kv4.h -- the paged 4-bit KV cache: page layout and launchers (kv4.hip,
// kv4_attn.hip, kv_plan.hip).  All pointers are device pointers.
//
// A value is code * scale: the code E2M1 (0, .5, 1, 1.5, 2, 3, 4, 6 and a
// sign, the element that gfx950 converts to f16 in one instruction per two),
// the scale an f16 of 9 significant bits per 32 values, so that every value
// is exactly an f16 number (2 + 9 <= 11 bits; scales are multiples of 2^-23,
// so the halves of the smallest are multiples of 2^-24).
//
// A page holds `ps` tokens (16 .. 256, a power of two) of every KV head.  Per
// head, in this order:
//   K codes  [ps][hd/2]         byte j of a row: dims 2j (low), 2j + 1 (high)
//   V codes  [ps/16][hd/2][16]  byte (b*16 + a, token): dims b*32 + a (low),
//                               b*32 + 16 + a (high)
//   K scales [ps][hd/32] f16
//   V scales [ps/16][hd/32][16 tokens] f16
// V is stored token-minor: the product of the probabilities with V runs over
// tokens, and a lane of its matrix operand holds consecutive tokens of one
// dim.  No byte is shared by two tokens, so appends never read.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace draco {

struct Kv4View {
    uint8_t* data;
    unsigned page_bytes;  // n_kv * head_bytes (4096 heads of 256 tokens of 256 dims: 302 MB at most)
    int head_bytes;       // ps * (hd + hd / 8)
    int n_pages, ps_shift, n_kv, hd;
};

inline size_t kv4_head_bytes(int ps, int hd) { return (size_t)ps * (hd + hd / 8); }

struct Kv4AppendArgs {
    Kv4View c;
    const void *q, *k, *v;
    void* q_out;
    long q_stride, q_out_stride, k_stride, v_stride;  // elements per token
    const int* slot;
    int n_tok, n_head;
    int rot, n_axes;   // rot 0: no rotation
    const int* pos;    // [n_axes][pos_stride]
    long pos_stride;
    const float* table;  // [table_rows][rot/2][cos, sin]
    int table_rows;
    uint32_t axis[8];    // of pair i: bits 2 (i % 16) .. of word i / 16
    int kv_passes;       // (filled by kv4_append)
};
// Blocks of 256 threads of a launch, at most: it has fewer than 2^32 threads.
constexpr long KV4_MAX_GRID = 0xFFFFFF;
struct Kv4AppendGrid {
    long kv, blocks;  // blocks that write K and V, all
    int kv_passes;
};
Kv4AppendGrid kv4_append_grid(const Kv4AppendArgs& a);
long kv4_read_grid(const Kv4View& c, int n);
int kv4_append(Kv4AppendArgs a, bool f16, bool halves, hipStream_t st);
int kv4_read(const Kv4View& c, const int* slot, int n, float* k, float* v, hipStream_t st);

struct Kv4AttnArgs {
    Kv4View c;
    const void* q;
    void* out;
    long q_stride, out_stride;
    const int *cu_q, *kv_len, *block_table;
    int n_seq, n_tok, n_head, group, max_blocks;
    int window, sink;
    float scale_log2;  // scale * log2(e)
    int chunk;           // units of 64 keys a block takes at least
    int* count;          // per block: of the tile that it leaves unfinished, blocks that are done; 0 between calls
    float* part;         // two slots a block: [rows of a tile][hd + 4]; behind them the join's records
    unsigned part_bytes; // of the slots
    bool whole;          // a tile per block instead (no counters, no partial rows)
};
constexpr int KV4_MAX_BLOCKS = 4096;
constexpr size_t KV4_COUNT_BYTES = KV4_MAX_BLOCKS * sizeof(int);
struct Kv4AttnPlan {
    int rows;            // of a tile: 16 and 32 the decode kernel's, else the prompt kernel's
    bool whole;
    long grid;
    int chunk;
    size_t part_bytes, work;  // bytes of partial rows, of workspace
};
Kv4AttnPlan kv4_attn_plan(int hd, bool f16, int n_seq, int n_tok, int n_head, int n_kv, int max_q, long max_keys,
                          int cus);
size_t kv4_attn_workspace(int hd, int cus);  // enough for any of its plans
int kv4_attn(Kv4AttnArgs a, bool f16, const Kv4AttnPlan& p, void* work, hipStream_t st);

struct KvPlanArgs {
    int n_seq, max_blocks, n_pages, ps_shift, n_tok;
    int* block_table;
    const int *kv_len, *q_len, *free_list, *n_free;
    int *cu_q, *pos, *slot, *kv_len_out, *n_free_out, *status, *ticket;
};
int kv_plan(const KvPlanArgs& a, hipStream_t st);
struct KvReleaseArgs {
    int n_seq, max_blocks, n_pages, ps_shift;
    const int* block_table;
    int* block_table_out;
    const int *kv_len, *keep;
    int* free_list;
    const int* n_free;
    int *kv_len_out, *n_free_out, *ticket;
};
int kv_release(const KvReleaseArgs& a, hipStream_t st);

}  // namespace draco
