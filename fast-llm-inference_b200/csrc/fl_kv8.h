// Private to the 8-bit paged KV cache sources (kv8.cu, kv8_attn.cu): the
// handle, the device tables of a plan and the layout of the codes.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <vector>

#include "fl_cuda.h"
#include "fl_kernels.h"

namespace fl {

constexpr int kKv8Block = FL_KV8_BLOCK;           // positions per scale
constexpr int kKv8Sub = kPageSize / kKv8Block;    // scales per page and head
constexpr int kKv8Long = 256;                     // packed query rows that a CTA of the prefill kernel takes

// Codes of one (page, kv head) are kPageSize * head_dim bytes: per block of
// 16 positions, per chunk of 32 dimensions, 512 bytes in the order in which a
// warp's lanes feed them to mma.m16n8k16, 16 bytes a lane, so that a block
// is read with one coalesced 16-byte load per lane and chunk, straight into
// the registers that the products use:
//   K, lane 4 n + t: 8 dimensions 8 t .. 8 t + 7 of the two positions
//      4 (n >> 1) + (n & 1) and that + 2 (the columns n of the two 8-wide
//      score tiles of the block)
//   V, lane 4 c + t: the 4 dimensions 4 c .. 4 c + 3, each for the four
//      positions 4 t .. 4 t + 3 (the probabilities that lane t of a row holds)
// INT8 codes are stored offset by 128, so that byte u under 0x64 is the half
// 1024 + u and the value is that less 1152, exact.

// Counts and constants that a plan leaves on the device.
struct Kv8Meta {
    int seqs, rows, units, gblocks;
    int refused;             // the plan changed nothing
    int pad;
    // the attention's two lists, of sequences with few and with many packed
    // query rows (new rows x group): per kv head
    struct List {
        long long tiles, work;   // row tiles, (row tile, page) pairs
        long long max_pages;     // of one of its sequences
    } list[2];
};

// Device arrays of a plan (all owned by the handle).
struct Kv8Tables {
    int *block_table, *held, *free_pages, *n_free, *row_start, *kv_start, *slot, *pos, *row_seq, *status;
    int *ctx;          // [max_seqs] cached positions of the planned sequences
    int *take_start, *rel_start, *unit_start, *gblk_start;  // [max_seqs + 1]
    long long *tile_start[2], *work_start[2];   // [max_seqs + 1] of each list: tiles and pairs before a sequence
    int *unit_row;     // [max_rows] first row of every (sequence, 16-position block) touched
    Kv8Meta* meta;
};

}  // namespace fl

struct fl_kv8 {
    fl_kv8_config_t c;
    int device = 0, sms = 148;
    int max_pages = 0;          // pages per sequence
    int group = 1, tile_rows = 16;
    int parts[2] = {};          // CTAs of an attention launch, of either list's kernel
    int max_new = 0;            // bound of the last plan
    int captured_max_new = 0;   // of all plans captured into graphs, which may be replayed at any time
    unsigned long long plan_capture = 0;   // the capture that the last plan went into, 0: none
    int nseq = 0;
    std::vector<void*> bufs;
    std::vector<uint8_t*> k, v;       // [layers] codes
    std::vector<float*> ks, vs;       // [layers] scales
    fl::Kv8Tables t = {};
    float* part[2] = {};        // [2 parts][rows of a tile][head_dim] partial outputs
    float2* part_ml[2] = {};    // [2 parts][rows of a tile] (maximum, sum)
    int* part_cnt[2] = {};      // [parts] arrivals, zero between launches
    float4* fold = nullptr;     // [parts[1]][head_dim / 4][kKv8Long] sums over a CTA's earlier pages
};

namespace fl {

struct Kv8AttnParams {
    const uint8_t *k, *v;
    const float *ks, *vs;
    Kv8Tables t;
    int max_pages, heads, kv_heads, group, head_dim, type, dtype;
    const void* q;
    void* out;
    size_t ldq, ldo;
    int rows;            // rows of q and out
    float scale;         // of the scores, times log2(e)
    const uint8_t* mask; // [rows][ldm] or null: causal
    int ldm;
};
// One list's tiles and the workspace of its kernel.
struct Kv8Tiles {
    int list;
    const long long *tile_start, *work_start;
    float* part;
    float2* part_ml;
    int* part_cnt;
    float4* fold;        // the prefill kernel's sums over earlier pages
    // the prefill kernel's bounded waits; fail_at > 0: the issuing thread of CTA
    // fail_cta stops before its fail_at-th group of products, as if a wait had run out
    long long wait_clocks;
    int fail_cta, fail_at;
};
constexpr long long kKv8WaitClocks = 4000000000ll;   // about 2 s
cudaError_t launch_kv8_attention(const Kv8AttnParams& p, const Kv8Tiles& tl, int ctas, cudaStream_t s);
cudaError_t launch_kv8_prefill(const Kv8AttnParams& p, const Kv8Tiles& tl, int ctas, cudaStream_t s);
// CTAs of the attention kernel that one SM holds (for the plan's split).
int kv8_attention_occupancy(int head_dim, int type, int dtype);
cudaError_t kv8_prefill_prepare(int head_dim, int type, int dtype);
int take_kv8_error();   // returns and clears the prefill kernel's error word

}  // namespace fl
