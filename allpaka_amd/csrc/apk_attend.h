// What the host (apk_host.cpp) and the attention kernels (kernels/attend.hip.h) share: the argument block and the layout of
// the scratch.
#pragma once
#include <stdint.h>

// Rows of a tile of the chunk kernel: flat (token, head of the group) rows of one kv head.  (The kernel for few rows takes
// 16.)
#define APK_ATT_CHUNK_ROWS 128u
// The scratch: one word, the number of tiles listed; from word 16 on 8 words for each of them (first row and rows of the
// sequence, tile, parts, slots of the first and the second part and the step to the next ones); from APK_ATT_PART_AT bytes
// on the parts' results, (tile_rows x (hd + 2)) floats per slot and kv head.
#define APK_ATT_MAX_LIST 32000u
#define APK_ATT_PART_AT (1u << 20)

struct apk_attend_args {
    const void* q;            // [rows][n_q * hd] of the activation type
    const void* k;            // fp16 [n_pages * page][n_kv * hd]
    const void* v;
    void* out;                // [rows][n_q * hd]
    const uint32_t* table;    // [n_seq][max_pages]
    const uint32_t* q_off;    // [n_seq + 1], or NULL: one row per sequence
    const uint32_t* kv_len;   // [n_seq]
    uint32_t* scratch;
    uint32_t* fault;
    uint32_t n_seq, rows, n_q, n_kv, hd, group;  // group = n_q / n_kv
    uint32_t page, page_magic, max_pages, n_pages;
    uint32_t window;          // 0: none
    uint32_t heads;           // kv heads that a workgroup takes (few rows: a power of two that divides n_kv; chunks: 1)
    uint32_t target;          // chunks: tiles are cut until about this many workgroups have work; few rows: workgroups per block of heads
    uint32_t unit_min;        // fewest units worth a part of their own
    uint32_t whole_units;     // few rows: not 0: every tile counts as this many units, and a piece is one tile
    uint32_t list_tiles;      // few rows: 1: the list has a place for every tile; 0: one for every workgroup
    uint32_t join_rows;       // rows that a workgroup of the joining launch takes
    uint32_t tile_rows, unit; // rows of a tile and keys of a unit, powers of two, and their logarithms
    uint32_t tile_shift, unit_shift;
    float scale;              // its magnitude
    float sign;               // and its sign, applied to q
    float c;                  // scale * log2(e), kept a normal number: what fp16 rows' products are multiplied by
};
