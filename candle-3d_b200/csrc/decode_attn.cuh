// Attention of a few rows over many keys, shared by l3d_paged_attention (keys in pages) and l3d_cross_attention
// (packed keys, equal groups of few rows).
#pragma once
#include "common.cuh"

namespace l3d {
namespace decode {

struct Params {
  int B, N, G, Hkv;             // N rows a sequence, query heads h G .. h G + G - 1 read key head h
  const char* q;
  char* out;
  int64_t qb, qn, qh, ob, on, oh;   // element strides
  const char *k, *v;
  int64_t ks[3], vs[3];         // strides of page, slot, head (packed: unused, row, head)
  int keys;                     // pages, or packed rows
  int size, width;              // tokens of a page, pages of a request (packed: size 0)
  const int32_t* table;
  int64_t table_stride;
  const void* lengths;          // paged: [B]; packed: offsets [B + 1]
  int len64, causal;
  float scale_log2;             // softmax scale * log2(e), > 0
  int tiles, rows;              // row tiles of a key head, rows of a tile's part
  int total_warps;
  int* starts;                  // workspace: key tiles before each sequence [B + 1]
  float *part_l, *part_o;       // [2 warps, rows], [2 warps, rows, D]
};

constexpr int MAX_BATCH = 4096;
// Workspace bytes, the same for every division of the keys; 0: nothing to do.
size_t workspace_size(int64_t B, int64_t N, int64_t G, int64_t Hkv, int64_t longest, int64_t D);
// Fills in tiles, rows, total_warps and the workspace's places, and launches.  `longest`: the most keys a
// sequence can have.
cudaError_t launch(Params p, bool f16, int D, int64_t longest, void* workspace, cudaStream_t s);

}  // namespace decode
}  // namespace l3d
