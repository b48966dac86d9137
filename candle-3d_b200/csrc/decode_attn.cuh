// Attention of a few rows over many keys, shared by l3d_paged_attention (keys in pages) and l3d_cross_attention
// (packed keys, equal groups of few rows).
#pragma once
#include "common.cuh"

namespace l3d {
namespace decode {

// How a K or V map [pages, slots, heads, D] lists its dimensions.
struct View {
  int hn, hm;                   // heads before slots; 0: heads expanded (stride 0)
};
// K and V as the caller has them: element strides of page, slot, head (packed: of row and head).
struct Keys {
  const void *k, *v;
  int64_t ks[3], vs[3];
  int64_t D;
};

struct Params {
  int B, N, G, Hkv;             // N rows a sequence, query heads h G .. h G + G - 1 read key head h
  const char* q;
  char* out;
  int64_t qb, qn, qh, ob, on, oh;   // element strides
  View kw, vw;
  int keys;                     // pages, or packed rows
  int size, width;              // tokens of a page, pages of a request (packed: size 0)
  int box;                      // rows of a load: the largest power of two, up to a tile's keys, that divides the size
  int box_bytes;                // what a load of K and V brings (failure self-test: 16 more, which never come)
  uint32_t mul;                 // j / size = (j * mul) >> (32 + shift), j < 2^30 (size > 1)
  int shift;
  const int32_t* table;
  int64_t table_stride;
  const void* lengths;          // paged: [B]; packed: offsets [B + 1]
  int len64, causal;
  float scale_log2;             // softmax scale * log2(e), > 0
  int height, tiles, rows;      // rows of a row tile, row tiles of a key head, rows of a tile's part
  int total_warps;              // 0: a block for each head and row tile
  uint64_t wait_ns;
  int* starts;                  // workspace: key tiles before each sequence [B + 1],
  int4* edges;                  // the item divided at the end of each warp's stretch [warps], where items outnumber warps,
  float *part_l, *part_o;       // [2 warps, rows], [2 warps, rows, D]
};

constexpr int MAX_BATCH = 4096;
// Workspace bytes, whatever the lengths are; 0: none needed.
size_t workspace_size(int64_t B, int64_t N, int64_t G, int64_t Hkv, int64_t longest, int64_t D);
// Fills in what follows from the sizes and the workspace, and launches; an entry's status.  `longest`: the most
// keys a sequence can have.  timeout_ns: 0, or the failure self-test, in which every wait for a load runs out then.
int launch(const char* op, Params p, const Keys& kv, bool f16, int64_t longest, void* workspace, cudaStream_t s,
           uint64_t timeout_ns = 0);

}  // namespace decode
}  // namespace l3d
