// kr_kv.h -- operators over a caller's paged key / value cache (krasis_amd.kv_cache.PagedKVCache): what the entry points in kr_kv.cpp hand to the kernels in kr_kv_store.hip
// (rows quantised into the pages, read back, moved), kr_kv_step_dev.h and kr_kv_tile_dev.h (attention over the pages) and kr_kv_join.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/krasis_hip.h"

struct KvDiv { uint32_t d, magic; };      // a divisor and floor(2^32 / d), at most 2^32 - 1
inline KvDiv kv_divisor(uint32_t d) { return KvDiv{d, d == 1 ? 0xFFFFFFFFu : (uint32_t)((1ull << 32) / d)}; }

// one layer's pages: keys / values [slots][kv_heads][dim] in the page format, scales [slots][kv_heads][dim / 32] for the microscaled ones; slot = page * page_tokens + offset
struct KvPages {
    uint8_t *k, *v, *ks, *vs;
    int row_bytes, srow_bytes;         // bytes of a slot: all heads' codes / scales
    int head_bytes, shead_bytes;       // bytes of one head of a slot
    uint32_t row16;                    // row_bytes / 16: places in the pages are counted in units of 16 bytes
    uint32_t scale_and, scale_or;      // (scale byte & scale_and) | scale_or: pages of plain E4M3 give any byte of theirs, which becomes 127
    int scale_shift;                   // place in the pages >> scale_shift = place of its scales
    KvDiv page;                        // tokens
};
// the sequences of a step, on the device
struct KvSeqs {
    const int *row0, *lens, *page0, *pages, *slots;      // [batch + 1] first new row, [batch] stored tokens with the new ones, [batch] first entry in pages, page ids, [rows] slots of the new rows
    int batch, rows;
};

struct KvRowsArgs { KvPages p; const int* slots; void *k, *v; long k_tok, k_head, v_tok, v_head; KvDiv per_row, per_head; int rows, format, half; };      // strides in elements; per_row, per_head: units of eight channels; half: rows are f16
struct KvMoveArgs { uint8_t* base[4]; long layer_bytes[4]; int row_bytes[4]; const int *start, *src, *dst; int n_seq, layers; };

struct KvAttnArgs {
    KvPages p;
    KvSeqs s;
    const uint16_t* q; uint16_t* out;
    long q_tok, q_head;                // strides in elements; out is [rows][heads][dim]
    const int* parents;                // drafted trees: parent draft of every new row, or NULL
    int heads;
    KvDiv kv_heads, G;                 // G = heads / kv_heads
    int window, first;
    float scale_log2;                  // scale * log2(e): scores are kept in units of log 2
    int min_rows, max_rows;            // the sequences of this launch: those whose new rows times G lie in between
    KvDiv tps;                         // key tiles a workgroup takes at most
    int items, whole, one;                    // whole: items / (8 kv_heads) * (8 kv_heads); one: no sequence of this launch has more than one new token, and there are no trees
    float* ws;                         // partial results of sequences that are split: [item][rows][dim] sums, then [item][rows][2] reference (kr_kv_dev.h) and denominator
};

int kr_launch_kv_write(const KvRowsArgs& a, hipStream_t st);
int kr_launch_kv_read(const KvRowsArgs& a, hipStream_t st);
int kr_launch_kv_move(const KvMoveArgs& a, hipStream_t st);
// by the width of the pages' numbers; half: q and out are f16; waves: of a workgroup, 32 rows each
int kr_launch_kv_step_16(const KvAttnArgs& a, int dim, int half, hipStream_t st);
int kr_launch_kv_step_8(const KvAttnArgs& a, int dim, int half, hipStream_t st);
int kr_launch_kv_step_4(const KvAttnArgs& a, int dim, int half, hipStream_t st);
int kr_launch_kv_tile_16(const KvAttnArgs& a, int dim, int half, int waves, hipStream_t st);
int kr_launch_kv_tile_8(const KvAttnArgs& a, int dim, int half, int waves, hipStream_t st);
int kr_launch_kv_tile_4(const KvAttnArgs& a, int dim, int half, int waves, hipStream_t st);
int kr_launch_kv_join(const KvAttnArgs& a, int dim, int bm, int kt, int units, int few, int half, hipStream_t st);
constexpr int KV_MAX_SHARES = 1024;                  // of a row tile

constexpr int KV_STEP_BM = 16, KV_STEP_KT = 32;      // rows (new tokens x heads of a group) and keys of a tile in kr_kv_step_dev.h
constexpr int KV_TILE_KT = 64;                       // keys of a tile in kr_kv_tile_dev.h; 32 rows a wave
// Waves that a SIMD holds of the latter, by measurement.  Heads of 64 channels take three under bf16 queries over eight and four bits, though 4 and 8 registers do not fit into 168: two prompts
// of 8192 and 3001 tokens 405 -> 382 us.  Others would spill more: 16-bit pages 390 us with two, 498 with three, f16 queries over eight bits 595 and 690.
// Of 128 channels (four waves a workgroup) f16 queries over eight bits take one: 64 sequences' drafts 96 us with one, 122 with two; over four bits 96 and 82, 16-bit pages, of which 7 registers
// spill, 82 and 79.  Eight waves a workgroup are two a SIMD: 5 registers of f16 queries over four bits spill.
__host__ __device__ constexpr int kv_tile_waves(int dim, int fmt, bool half) {
    return dim == 64 && fmt != 0 && !half ? 3 : dim < 128 || (dim == 128 && !(fmt == 1 && half)) ? 2 : 1;
}
// Waves of a workgroup in kr_kv_step_dev.h, one workgroup a CU.  one: every sequence has one new token: as many as the registers hold (half: f16 queries, two pieces over pages that become bf16).
// Several new tokens take 8, and 4 from 192 channels on; by their registers they could take more (64 channels 128 to 142, 128 channels 158 to 193), which is not measured.
// (Of 96 channels 16-bit pages take twelve: with sixteen two registers spill, 32 requests of up to 8192 tokens 57.4 us, 53.8 with twelve.)
__host__ __device__ constexpr int kv_step_waves(int dim, int fmt, bool half, bool one) {
    return !one ? (dim <= 128 ? 8 : 4) : dim == 64 || (dim == 128 && fmt == 2 && !half) ? 16 : dim <= 128 ? 12 : dim == 256 && fmt == 0 ? 4 : 8;
}
constexpr int KV_MAX_TREE = 64;                      // drafts of one sequence: their ancestors are a 64-bit word

// ---- the division of a launch into items, the same on the host (how many) and on the device (which one)
// key tiles that any row tile of a sequence can need; BM rows and KT keys a tile
__host__ __device__ inline int kv_tiles_ub(int len, int cnt, KvDiv G, int window, int first, bool tree, int bm, int kt) {
    const int all = (len + kt - 1) / kt;
    if (window <= 0) return all;
    const long span = (long)window + (tree ? cnt : (int)(((uint64_t)(bm - 1) * G.magic) >> 32) + 2);      // tokens from the first row's window to the last row, or one more
    const int some = (int)((span < len ? span : len) / kt) + 2 + (first + kt - 1) / kt;
    return some < all ? some : all;
}
__host__ __device__ inline int kv_row_tiles(int cnt, int G, int bm) { return (cnt * G + bm - 1) / bm; }
