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

// How the packed product over the shared prefix is cut (cdr_tile_attention.cu).
struct PackedPlan {
  int seqs_per_half, row_tiles, split_blocks, splits;
  int ctas;            // SMs it takes; the streaming kernel behind it runs on the others
  float us;            // estimated time of both
};

// How the keys of few query rows are streamed (cdr_cache_attention.cu).
struct StreamPlan {
  int m_tiles, ctas, n_warps, rows_cap, group, groups;
  int cluster;         // > 0: a cluster of so many CTAs per task, no scratch
  int64_t tasks, slots, units;     // units of 32 keys: the most there can be (every sequence at full length)
};

// The weights of a row are rounded to the input type for the second product (the matrix instructions take both operands in one
// 16-bit type): relative 2^-8 at most each at bf16, 2^-11 at f16, independent from key to key.  f16 ends at 2^-24, and
// against a dominating key the many weights of a long cache can all be smaller.  There the reference of the exponentials is
// the running maximum minus 7: the largest weight is 2^7 (2^15 before a rescale, below the type's 2^16) and weights count down
// to 2^-32.  Sums are taken against the same reference, so nothing else changes.
template <bool BF16>
struct WeightShift { static constexpr float value = BF16 ? 0.0f : 7.0f; };   // log2 units

// Many query rows (cdr_tile_attention.cu).  Their `ws` is kTileCounterBytes for the tile counter, 32-byte aligned.
constexpr size_t kTileCounterBytes = 256;
// prefix, sinks and window of every (sequence, query head), 256 queries per tile
int launch_tile_attention(const CacheAttn& a, void* ws, cudaStream_t stream);
float tile_attention_us(const CacheAttn& a);   // estimated time
// the shared prefix alone, for G * Sq <= 128 query rows per sequence and key head, into *part in `ws`; `own_units`: of the
// streaming kernel that runs beside it
PackedPlan plan_packed(const CacheAttn& a, int64_t own_units);
size_t packed_workspace(const CacheAttn& a, const PackedPlan& plan);
int launch_packed_prefix(const CacheAttn& a, const PackedPlan& plan, void* ws, PrefixPartials* part, cudaStream_t stream);

#ifdef __CUDACC__
__device__ __forceinline__ int sequence_length(const CacheAttn& a, int b) {
  if (!a.lengths) return a.Skv;
  const int64_t n = a.lengths_i64 ? __ldg(static_cast<const long long*>(a.lengths) + b)
                                  : static_cast<int64_t>(__ldg(static_cast<const int*>(a.lengths) + b));
  return n < 0 ? 0 : n > a.Skv ? a.Skv : static_cast<int>(n);
}
#endif

}  // namespace cdr
