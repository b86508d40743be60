// What the host (apk_host.cpp) and the attention kernels (kernels/attend.hip.h) share: the argument block and the tile sizes.
#pragma once
#include <stdint.h>

// Rows of one tile of the chunk kernel (flat (token, head of the group) rows of one kv head), keys of one unit of work
// of each kernel, and query heads of one tile of the single-token kernel.
#define APK_ATT_CHUNK_ROWS 128u
#define APK_ATT_CHUNK_UNIT 64u
#define APK_ATT_TOKEN_UNIT 128u
#define APK_ATT_TOKEN_ROWS 16u

struct apk_attend_args {
    const void* q;            // [rows][n_q * hd] of the activation type
    const void* k;            // fp16 [n_pages * page][n_kv * hd]
    const void* v;
    void* out;                // [rows][n_q * hd]
    const uint32_t* table;    // [n_seq][max_pages]
    const uint32_t* q_off;    // [n_seq + 1], or NULL: one row per sequence
    const uint32_t* kv_len;   // [n_seq]
    float* part;              // partial results of tiles whose keys are split: slots of (rows x (hd + 2)) floats
    uint32_t* fault;
    uint32_t n_seq, rows, n_q, n_kv, hd, group;  // group = n_q / n_kv
    uint32_t page, page_magic, max_pages, n_pages;
    uint32_t window;          // 0: none
    uint32_t head_tiles;      // tiles of query heads per kv head (single-token kernel; 1 for chunks)
    uint32_t target;          // tiles are split until about this many workgroups have work; at most 2 * target slots are used
    uint32_t unit_min;        // fewest units worth a part of their own
    uint32_t tile_rows, unit; // rows and keys of the kernel's tile (the constants above)
    float c;                  // |scale| * log2(e), kept above zero
    float sign;               // the sign of scale, applied to q
};
