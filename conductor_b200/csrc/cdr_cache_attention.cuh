// The two attentions over a key/value cache (window_attention, prefix_attention), seen by their
// kernels as one problem:
//
//   query row i of sequence b stands at position p = L_b - Sq + i of the sequence's own keys, where
//   L_b = clamp(lengths[b], 0, Skv).  It sees
//     - every key of the shared prefix (P keys per key head, P = 0 without one) and
//     - own key j when  j <= p  and  (j > p - window  or  j < sinks).
//   A row with p < 0 (a batch padded to Sq queries) sees nothing and its output is 0.
//
// Heads are grouped: query heads h*G .. h*G + G-1 share key head h.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "cdr_common.cuh"

namespace cdr {

// element strides of one [B, H, S, D] operand (D contiguous)
struct HeadStrides {
  int64_t b, h, s;
};

struct CacheAttn {
  const void *q, *k, *v, *pk, *pv;
  void* out;
  const void* lengths;  // [B] i32 / i64, or nullptr: every sequence uses all Skv keys
  int lengths_i64;
  HeadStrides sq, sk, sv, spk, spv, so;
  int B, Hq, Hkv, G, Sq, Skv, P, D;
  int window, sinks;    // clamped to 2^30: positions are below that
  float scale_log2;     // scale * log2(e)
  int bf16;
};

// Partial results of the shared prefix, one per key split and packed query row, in caller scratch:
// O already divided by its sum, and log2 of the sum of exponentials (base 2, scaled scores).
struct PrefixPartials {
  const float* o;      // [splits][Hkv][rows][D]
  const float* lse;    // [splits][Hkv][rows]
  int splits;          // 0: none
  int rows;            // packed rows: 128 per group of `seqs` sequences
  int seqs;

  // row of query i, head gi of its group, sequence b; its part n is at (n * Hkv + hkv) * rows + row
  __host__ __device__ __forceinline__ int row_of(const CacheAttn& a, int b, int i, int gi) const {
    const int group = b / seqs;
    return group * 128 + ((b - group * seqs) * a.G + gi) * a.Sq + i;
  }
};

// Few query rows per key head: the keys are streamed once (cdr_cache_attention.cu).  part.splits > 0: joined with
// the partial results (launched right behind the kernel that makes them); else the prefix is streamed as well.
int launch_stream_attention(const CacheAttn& a, const PrefixPartials& part, void* ws, cudaStream_t stream);
size_t stream_workspace(const CacheAttn& a, bool behind_prefix);   // 16-byte aligned start
float stream_units(const CacheAttn& a);        // 16 KB (D = 128) pieces of own keys, at full lengths

// Many query rows (cdr_tile_attention.cu).  `ws` starts with kTileCounterBytes for the tile counter.
constexpr size_t kTileCounterBytes = 256;
// prefix, sinks and window of every (sequence, query head), 256 queries per tile
int launch_tile_attention(const CacheAttn& a, void* ws, cudaStream_t stream);
// the shared prefix alone, for G * Sq <= 128 query rows per sequence and key head, into *part in `ws`
int launch_packed_prefix(const CacheAttn& a, void* ws, PrefixPartials* part, cudaStream_t stream);
size_t packed_workspace(const CacheAttn& a);   // with the counter; 32-byte aligned start
int packed_ctas(const CacheAttn& a);           // SMs it takes; the streaming kernel behind it runs on the others

#ifdef __CUDACC__
__device__ __forceinline__ int sequence_length(const CacheAttn& a, int b) {
  if (!a.lengths) return a.Skv;
  const int64_t n = a.lengths_i64 ? __ldg(static_cast<const long long*>(a.lengths) + b)
                                  : static_cast<int64_t>(__ldg(static_cast<const int*>(a.lengths) + b));
  return n < 0 ? 0 : n > a.Skv ? a.Skv : static_cast<int>(n);
}
#endif

}  // namespace cdr
