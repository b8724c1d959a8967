// K7 -- attention over a key/value cache for few query rows (decode and verification steps):
//   O = softmax(scale * Q K^T [window + sinks, cache length]) V
// for the G * Sq query rows that share one key head of one sequence, and the entry points of
// CDR_T_WINDOW_ATTENTION and CDR_T_PREFIX_ATTENTION.  The reference has no attention over a cache;
// its kernels (choreo-op/attention-gcu-only-test.co:15-134) take q, k and v of one length.
//
// HBM bound: every visible key and value is read once for the (at most 16) rows of a task.  The
// keys of a task are split over the warps of a thread-block cluster (4 warps per CTA, 1 to 16 CTAs),
// each warp running the online-softmax recurrence over blocks of 16 keys on its own:
//   - K and V go from global memory straight into the operand registers of m16n8k16 matrix
//     instructions.  The order of the contraction index is free as long as both operands use the
//     same one, so a thread takes 16 contiguous bytes of a K row (and of the Q row) for two
//     k-steps; for P V it takes 16 bytes of four V rows and pairs them with byte permutes.  No
//     shared memory, no barrier in the loop.  16 rows are the instruction's height: a task with
//     fewer rows pays nothing for it, the loads set the pace.
//   - the K registers are reloaded for the next block right behind the score products, the V
//     registers behind the output products: a warp keeps 4 to 8 KB in flight (HD = 128).
//   - the accumulator is rescaled only when a row's maximum grew by more than 2^8; exact after the
//     final division because the sums use the same reference.
// The warps' (maximum, sum, O) are joined in shared memory, the CTAs' through distributed shared
// memory, each CTA writing 16 / cluster-size rows: one launch, no scratch, no atomics, and the order
// of the sums is fixed.  P is rounded to the input type for the second product (relative 2^-9 per
// weight at bf16, independent per key); scores, maxima, sums and O stay in fp32.
#include <cuda.h>
#include <math.h>

#include "cdr_cache_attention.cuh"
#include "cdr_sm100.cuh"

namespace cdr {
namespace {

constexpr int SA_WARPS = 4;          // per CTA; they split the keys
constexpr int SA_ROWS = 16;          // query rows of a task (m of the matrix instruction)
constexpr int SA_KEYS = 16;          // keys per block (k of the second product)
constexpr int SA_MAX_CLUSTER = 16;
constexpr float SA_RESCALE = 8.0f;   // log2 units

struct StreamArgs {
  CacheAttn a;
  PrefixPartials part;
  int m_tiles;        // tasks per (sequence, key head)
  int cluster;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if (BF16) { __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<uint32_t*>(&t); }
  __half2 t = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&t);
}

// a cached key is read by the CTAs of one task (and of the other row tiles of its head) only
__device__ __forceinline__ uint4 ld_cache16(const unsigned char* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// The keys a task reads, as up to three ranges of blocks of 16: prefix, sinks, window.
struct KeyRanges {
  int n_prefix, n_sink, n_total;   // block counts (cumulative)
  int prefix_end, sink_end, lo, hi;
};

struct Block {
  const unsigned char *k, *v;      // row 0 of the source
  int64_t ks, vs;                  // row pitch in bytes
  int base, end;                   // first key, one past the last key that may be read
  int own;                         // the sequence's own keys (masked by position), not the prefix
};

template <int HD, bool BF16>
__global__ void __launch_bounds__(SA_WARPS * 32, 3) stream_attention_kernel(const __grid_constant__ StreamArgs args) {
  constexpr int KC = HD / 32;      // 16-byte chunks of a K row per thread
  constexpr int VC = HD / 64;      // 16-byte chunks of a V row per thread
  constexpr int PITCH = HD + 4;
  __shared__ __align__(16) float sm_o[SA_WARPS][SA_ROWS][PITCH];
  __shared__ float sm_m[SA_WARPS][SA_ROWS], sm_l[SA_WARPS][SA_ROWS];
  const CacheAttn& a = args.a;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int cs = args.cluster;
  const int rank = blockIdx.x % cs;            // == %cluster_ctarank: the cluster is 1-D along x
  int task = blockIdx.x / cs;
  const int mt = task % args.m_tiles; task /= args.m_tiles;
  const int hkv = task % a.Hkv, b = task / a.Hkv;

  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int len = sequence_length(a, b);
  const int off = len - a.Sq;                  // position of query 0
  const int rows = a.G * a.Sq;                 // row r = i * G + g: a tile spans few positions
  const int r_first = mt * SA_ROWS, r_last = min(r_first + SA_ROWS, rows) - 1;
  const int p_last = off + r_last / a.G;
  const int p_first = max(off + r_first / a.G, 0);   // first row of the tile that sees keys

  KeyRanges kr;
  kr.lo = kr.hi = kr.sink_end = kr.prefix_end = 0;
  if (p_last >= 0) {
    kr.hi = p_last + 1;
    kr.lo = max(p_first - a.window + 1, 0);
    kr.sink_end = min(a.sinks, kr.lo);
    if (args.part.splits == 0) kr.prefix_end = a.P;
  }
  kr.n_prefix = (kr.prefix_end + SA_KEYS - 1) / SA_KEYS;
  kr.n_sink = kr.n_prefix + (kr.sink_end + SA_KEYS - 1) / SA_KEYS;
  kr.n_total = kr.n_sink + (kr.hi - kr.lo + SA_KEYS - 1) / SA_KEYS;

  const unsigned char* k_own = static_cast<const unsigned char*>(a.k) + (b * a.sk.b + hkv * a.sk.h) * 2;
  const unsigned char* v_own = static_cast<const unsigned char*>(a.v) + (b * a.sv.b + hkv * a.sv.h) * 2;
  const unsigned char* k_pre = static_cast<const unsigned char*>(a.pk) + hkv * a.spk.h * 2;
  const unsigned char* v_pre = static_cast<const unsigned char*>(a.pv) + hkv * a.spv.h * 2;

  auto block_of = [&](int t) {
    Block x;
    if (t < kr.n_prefix) {
      x = Block{k_pre, v_pre, a.spk.s * 2, a.spv.s * 2, t * SA_KEYS, kr.prefix_end, 0};
    } else if (t < kr.n_sink) {
      x = Block{k_own, v_own, a.sk.s * 2, a.sv.s * 2, (t - kr.n_prefix) * SA_KEYS, kr.sink_end, 1};
    } else {
      x = Block{k_own, v_own, a.sk.s * 2, a.sv.s * 2, kr.lo + (t - kr.n_sink) * SA_KEYS, kr.hi, 1};
    }
    return x;
  };

  // this thread's two query rows: g and g + 8 of the tile
  int pos[2];
  uint4 qf[2][KC];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r_first + g + 8 * h;
    pos[h] = -1;
    const bool live = r <= r_last;
    if (live) pos[h] = off + r / a.G;
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      qf[h][j] = make_uint4(0, 0, 0, 0);
      if (live) {
        const int64_t e = b * a.sq.b + static_cast<int64_t>(hkv * a.G + r % a.G) * a.sq.h + static_cast<int64_t>(r / a.G) * a.sq.s;
        qf[h][j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(a.q) + e * 2 + j * 64 + c * 16));
      }
    }
  }

  uint4 kf[2][KC], vf[4][VC];
  // keys beyond the range's end are read from its last key instead and masked
  auto load_k = [&](const Block& x) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const unsigned char* p = x.k + min(x.base + n * 8 + g, x.end - 1) * x.ks + c * 16;
#pragma unroll
      for (int j = 0; j < KC; ++j) kf[n][j] = ld_cache16(p + j * 64);
    }
  };
  auto load_v = [&](const Block& x) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const unsigned char* p = x.v + min(x.base + (n >> 1) * 8 + 2 * c + (n & 1), x.end - 1) * x.vs + g * 16;
#pragma unroll
      for (int j = 0; j < VC; ++j) vf[n][j] = ld_cache16(p + j * 128);
    }
  };

  float o[VC][8][4];
#pragma unroll
  for (int j = 0; j < VC; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][e][i] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  // a CTA takes a contiguous share of the blocks, its warps take them in turn
  const int per = (kr.n_total + cs - 1) / cs;
  const int t_end = min((rank + 1) * per, kr.n_total);
  int t = rank * per + warp;
  const bool one_position = p_first == p_last;   // every live row sees exactly the keys of the ranges
  Block x;
  if (t < t_end) {
    x = block_of(t);
    load_k(x);
    load_v(x);
  }
  for (; t < t_end; t += SA_WARPS) {
    const bool more = t + SA_WARPS < t_end;
    float s[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
    for (int j = 0; j < KC; ++j)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        mma16816<BF16>(s[n], qf[0][j].x, qf[1][j].x, qf[0][j].y, qf[1][j].y, kf[n][j].x, kf[n][j].y);
        mma16816<BF16>(s[n], qf[0][j].z, qf[1][j].z, qf[0][j].w, qf[1][j].w, kf[n][j].z, kf[n][j].w);
      }
    const Block cur = x;
    if (more) {
      x = block_of(t + SA_WARPS);
      load_k(x);
    }

    // scores in log2 units; s[n][2h + e] belongs to row g + 8h and key base + 8n + 2c + e
    const bool masked = cur.base + SA_KEYS > cur.end || (cur.own && !one_position);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = s[n][i] * a.scale_log2;
        if (masked) {
          const int key = cur.base + 8 * n + 2 * c + (i & 1), p = pos[i >> 1];
          if (key >= cur.end || (cur.own && (key > p || (key <= p - a.window && key >= a.sinks)))) v = -INFINITY;
        }
        s[n][i] = v;
      }
    float mx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
      mx[h] = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] + SA_RESCALE || mx[1] > m[1] + SA_RESCALE)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float m_new = fmaxf(m[h], mx[h]);
        const float f = m[h] == -INFINITY ? 0.0f : ex2(m[h] - m_new);
        m[h] = m_new;
        l[h] *= f;
#pragma unroll
        for (int j = 0; j < VC; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) { o[j][e][2 * h] *= f; o[j][e][2 * h + 1] *= f; }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float ref = m[h] == -INFINITY ? 0.0f : m[h];     // nothing seen yet: every weight is exp2(-inf) = 0
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = ex2(s[n][2 * h + e] - ref);
          s[n][2 * h + e] = p;
          l[h] += p;
        }
    }
    const uint32_t pa0 = pack16<BF16>(s[0][0], s[0][1]), pa1 = pack16<BF16>(s[0][2], s[0][3]);
    const uint32_t pa2 = pack16<BF16>(s[1][0], s[1][1]), pa3 = pack16<BF16>(s[1][2], s[1][3]);
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t v0 = (&vf[0][j].x)[w], v1 = (&vf[1][j].x)[w], v2 = (&vf[2][j].x)[w], v3 = (&vf[3][j].x)[w];
        mma16816<BF16>(o[j][2 * w], pa0, pa1, pa2, pa3, __byte_perm(v0, v1, 0x5410), __byte_perm(v2, v3, 0x5410));
        mma16816<BF16>(o[j][2 * w + 1], pa0, pa1, pa2, pa3, __byte_perm(v0, v1, 0x7632), __byte_perm(v2, v3, 0x7632));
      }
    if (more) load_v(x);
  }

  // ---- join the warps: o[j][e][2h + i] is row g + 8h, column 64 j + 8 (2c + i) + e
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (c == 0) { sm_m[warp][g + 8 * h] = m[h]; sm_l[warp][g + 8 * h] = l[h]; }
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<float4*>(&sm_o[warp][g + 8 * h][64 * j + 8 * (2 * c + i) + e]) =
              make_float4(o[j][e][2 * h + i], o[j][e + 1][2 * h + i], o[j][e + 2][2 * h + i], o[j][e + 3][2 * h + i]);
  }
  __syncthreads();
  if (cs > 1) {
    // the CTA's own result replaces warp 0's, where the other CTAs of the cluster read it
    constexpr int PER = SA_ROWS * HD / (SA_WARPS * 32);
    const int row = threadIdx.x / (HD / PER), d0 = threadIdx.x % (HD / PER) * PER;
    float mm = sm_m[0][row];
#pragma unroll
    for (int w = 1; w < SA_WARPS; ++w) mm = fmaxf(mm, sm_m[w][row]);
    float f[SA_WARPS], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < SA_WARPS; ++w) {
      f[w] = sm_m[w][row] == -INFINITY ? 0.0f : ex2(sm_m[w][row] - mm);
      sum += f[w] * sm_l[w][row];
    }
#pragma unroll
    for (int d = 0; d < PER; d += 4) {
      float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < SA_WARPS; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(&sm_o[w][row][d0 + d]);
        acc.x += f[w] * v.x; acc.y += f[w] * v.y; acc.z += f[w] * v.z; acc.w += f[w] * v.w;
      }
      *reinterpret_cast<float4*>(&sm_o[0][row][d0 + d]) = acc;
    }
    __syncthreads();                             // every reader of the warps' sums is done
    if (d0 == 0) { sm_m[0][row] = mm; sm_l[0][row] = sum; }
    sm100::cluster_sync_all();
  }

  // ---- rows of this CTA: join the parts (warps, or the cluster's CTAs) and the prefix's partial results
  const int n_parts = cs > 1 ? cs : SA_WARPS;
  const int rows_here = SA_ROWS / cs, vecs = HD / 8;
  for (int w = threadIdx.x; w < rows_here * vecs; w += SA_WARPS * 32) {
    const int row = rank * rows_here + w / vecs, d = w % vecs * 8;
    const int r = r_first + row;
    if (r > r_last) continue;
    const int i = r / a.G, hq = hkv * a.G + r % a.G;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sum = 0.0f;
    if (off + i >= 0) {
      auto part_ptr = [&](const float* p, int n) -> const float* {
        if (cs == 1) return p;
        return reinterpret_cast<const float*>(__cluster_map_shared_rank(p, n));
      };
      const int ws = cs > 1 ? 0 : 1;             // parts are warps of this CTA, or warp slot 0 of every CTA
      auto pm = [&](int n) { return *part_ptr(&sm_m[ws * n][row], n); };
      const size_t prow = (static_cast<size_t>(b) * a.Sq + i) * a.G + r % a.G;
      auto lse_of = [&](int n) { return __ldg(args.part.lse + (static_cast<size_t>(n) * a.Hkv + hkv) * args.part.rows + prow); };
      float mm = -INFINITY;
      for (int n = 0; n < n_parts; ++n) mm = fmaxf(mm, pm(n));
      for (int n = 0; n < args.part.splits; ++n) mm = fmaxf(mm, lse_of(n));
      for (int n = 0; n < n_parts; ++n) {
        const float mn = pm(n);
        if (mn == -INFINITY) continue;
        const float f = ex2(mn - mm);
        sum += f * *part_ptr(&sm_l[ws * n][row], n);
        const float* src = part_ptr(&sm_o[ws * n][row][d], n);
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 v = *reinterpret_cast<const float4*>(src + e);
          acc[e] += f * v.x; acc[e + 1] += f * v.y; acc[e + 2] += f * v.z; acc[e + 3] += f * v.w;
        }
      }
      for (int n = 0; n < args.part.splits; ++n) {
        const float ls = lse_of(n);
        if (ls == -INFINITY) continue;
        const float f = ex2(ls - mm);
        sum += f;
        const float* src = args.part.o + ((static_cast<size_t>(n) * a.Hkv + hkv) * args.part.rows + prow) * HD + d;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 v = __ldg(reinterpret_cast<const float4*>(src + e));
          acc[e] += f * v.x; acc[e + 1] += f * v.y; acc[e + 2] += f * v.z; acc[e + 3] += f * v.w;
        }
      }
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;     // no visible key: 0; NaN passes through
    uint32_t out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = pack16<BF16>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    const int64_t e0 = b * a.so.b + hq * a.so.h + static_cast<int64_t>(i) * a.so.s + d;
    *reinterpret_cast<uint4*>(static_cast<unsigned char*>(a.out) + e0 * 2) = make_uint4(out[0], out[1], out[2], out[3]);
  }
  if (cs > 1) sm100::cluster_sync_all();         // no CTA leaves while another still reads its part
}

// ---------------------------------------------------------------- host side
template <int HD, bool BF16>
int launch_stream_cfg(const StreamArgs& s, int64_t tasks, cudaStream_t stream) {
  auto kern = stream_attention_kernel<HD, BF16>;
  int dev = 0;
  CDR_CUDA_TRY(cudaGetDevice(&dev));
  static bool configured_dev[64] = {false};
  if (!configured_dev[dev & 63]) {
    CDR_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    configured_dev[dev & 63] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tasks * s.cluster), 1, 1);
  cfg.blockDim = dim3(SA_WARPS * 32, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(s.cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  CDR_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, s));
  return CDR_OK;
}

}  // namespace

int launch_stream_attention(const CacheAttn& a, const PrefixPartials& part, cudaStream_t stream) {
  StreamArgs s;
  s.a = a;
  s.part = part;
  const int64_t rows = static_cast<int64_t>(a.G) * a.Sq;
  s.m_tiles = static_cast<int>((rows + SA_ROWS - 1) / SA_ROWS);
  const int64_t tasks = static_cast<int64_t>(a.B) * a.Hkv * s.m_tiles;
  // Split a task over as many CTAs as keep the machine's 3 resident CTAs per SM busy, as long as every
  // warp gets two blocks of keys.
  int64_t keys = a.Skv < static_cast<int64_t>(a.window) + a.sinks + a.Sq ? a.Skv : static_cast<int64_t>(a.window) + a.sinks + a.Sq;
  if (part.splits == 0) keys += a.P;
  s.cluster = 1;
  while (s.cluster < SA_MAX_CLUSTER && tasks * s.cluster < 3 * sm_count() && keys > 2LL * SA_KEYS * SA_WARPS * s.cluster) s.cluster *= 2;
  if (tasks * s.cluster > 0x7fffffff) { set_error("attention: %lld row tiles are too many for one launch", (long long)tasks); return CDR_ERR_UNSUPPORTED; }
  if (a.D == 128) return a.bf16 ? launch_stream_cfg<128, true>(s, tasks, stream) : launch_stream_cfg<128, false>(s, tasks, stream);
  return a.bf16 ? launch_stream_cfg<64, true>(s, tasks, stream) : launch_stream_cfg<64, false>(s, tasks, stream);
}

// ---------------------------------------------------------------- entry points
namespace {

// [.., S, D] operand: D contiguous, every other stride a positive multiple of 16 bytes.  Extents of 1
// get a stride that the kernels may use for address arithmetic.
int check_operand(const cdr_tensor& t, const char* op, const char* name, int rank, int dtype, int64_t D, HeadStrides* st) {
  if (t.rank != rank) { set_error("%s: %s has rank %d, expected %d", op, name, t.rank, rank); return CDR_ERR_BAD_ARG; }
  if (t.dtype != dtype) { set_error("%s: %s differs from q in dtype", op, name); return CDR_ERR_BAD_ARG; }
  if (t.shape[rank - 1] != D) { set_error("%s: %s has head dimension %lld, q has %lld", op, name, (long long)t.shape[rank - 1], (long long)D); return CDR_ERR_BAD_ARG; }
  if (t.stride[rank - 1] != 1) { set_error("%s: the head dimension of %s must be contiguous", op, name); return CDR_ERR_UNSUPPORTED; }
  int64_t s[3] = {D, D, D};
  for (int i = 0; i < rank - 1; ++i) {
    if (t.shape[i] <= 1) continue;
    if (t.stride[i] <= 0 || t.stride[i] % 8 != 0 || t.stride[i] >= (1LL << 38)) {
      set_error("%s: stride %lld of %s is not a positive multiple of 8 elements", op, (long long)t.stride[i], name);
      return CDR_ERR_UNSUPPORTED;
    }
    s[i + 4 - rank] = t.stride[i];
  }
  *st = HeadStrides{s[0], s[1], s[2]};
  return CDR_OK;
}

int check_pointer(const void* p, int64_t n, const char* op, const char* name) {
  if (n == 0) return CDR_OK;
  if (!p) { set_error("%s: %s is a null pointer", op, name); return CDR_ERR_BAD_ARG; }
  if (!aligned16(p)) { set_error("%s: %s is not 16-byte aligned", op, name); return CDR_ERR_MISALIGNED; }
  return CDR_OK;
}

// Shapes, types, strides and pointers of (q, [prefix_k, prefix_v,] k, v[, lengths]) -> out.
int parse_problem(const char* op, const cdr_tensor* ins, int n_in, const cdr_tensor* outs, int n_out, bool prefix,
                  int has_lengths, float scale, CacheAttn* a, bool* empty) {
  const int want = 3 + (prefix ? 2 : 0) + (has_lengths ? 1 : 0);
  if (n_in != want || n_out != 1) { set_error("%s: expects %d inputs and 1 output, got %d and %d", op, want, n_in, n_out); return CDR_ERR_BAD_ARG; }
  const cdr_tensor &q = ins[0], &k = ins[prefix ? 3 : 1], &v = ins[prefix ? 4 : 2], &out = outs[0];
  if (q.rank != 4) { set_error("%s: q has rank %d, expected [batch, heads, queries, head dim]", op, q.rank); return CDR_ERR_BAD_ARG; }
  if (q.dtype != CDR_BF16 && q.dtype != CDR_F16) { set_error("%s: dtype %d unsupported (bf16 and f16 only)", op, q.dtype); return CDR_ERR_UNSUPPORTED; }
  const int64_t B = q.shape[0], Hq = q.shape[1], Sq = q.shape[2], D = q.shape[3];
  if (D != 64 && D != 128) { set_error("%s: head dim %lld unsupported (64 or 128)", op, (long long)D); return CDR_ERR_UNSUPPORTED; }
  if (!(scale > 0.0f) || !isfinite(scale)) { set_error("%s: scale must be positive and finite", op); return CDR_ERR_UNSUPPORTED; }
  if (int rc = check_operand(q, op, "q", 4, q.dtype, D, &a->sq)) return rc;
  if (int rc = check_operand(k, op, "k", 4, q.dtype, D, &a->sk)) return rc;
  if (int rc = check_operand(v, op, "v", 4, q.dtype, D, &a->sv)) return rc;
  if (int rc = check_operand(out, op, "the output", 4, q.dtype, D, &a->so)) return rc;
  const int64_t Hkv = k.shape[1], Skv = k.shape[2];
  for (int i = 0; i < 3; ++i)
    if (v.shape[i] != k.shape[i] || out.shape[i] != q.shape[i]) {
      set_error("%s: k and v, and q and the output, must have the same shapes", op);
      return CDR_ERR_BAD_ARG;
    }
  if (k.shape[0] != B) { set_error("%s: q has %lld sequences, k has %lld", op, (long long)B, (long long)k.shape[0]); return CDR_ERR_BAD_ARG; }
  if ((Hkv == 0) != (Hq == 0) || (Hkv && Hq % Hkv != 0)) {
    set_error("%s: %lld query heads cannot share %lld key heads", op, (long long)Hq, (long long)Hkv);
    return CDR_ERR_BAD_ARG;
  }
  int64_t P = 0;
  a->pk = a->pv = nullptr;
  a->spk = a->spv = HeadStrides{0, D, D};
  if (prefix) {
    const cdr_tensor &pk = ins[1], &pv = ins[2];
    if (int rc = check_operand(pk, op, "prefix_k", 3, q.dtype, D, &a->spk)) return rc;
    if (int rc = check_operand(pv, op, "prefix_v", 3, q.dtype, D, &a->spv)) return rc;
    P = pk.shape[1];
    if (pk.shape[0] != Hkv || pv.shape[0] != Hkv || pv.shape[1] != P) {
      set_error("%s: prefix_k and prefix_v must both be [%lld, prefix length, %lld]", op, (long long)Hkv, (long long)D);
      return CDR_ERR_BAD_ARG;
    }
    if (int rc = check_pointer(pk.data, numel(pk), op, "prefix_k")) return rc;
    if (int rc = check_pointer(pv.data, numel(pv), op, "prefix_v")) return rc;
    a->pk = pk.data;
    a->pv = pv.data;
  }
  a->lengths = nullptr;
  a->lengths_i64 = 0;
  if (has_lengths) {
    const cdr_tensor& n = ins[want - 1];
    if (n.dtype != CDR_I32 && n.dtype != CDR_I64) { set_error("%s: lengths must be int32 or int64", op); return CDR_ERR_BAD_ARG; }
    if (n.rank != 1 || n.shape[0] != B || !is_contiguous(n)) { set_error("%s: lengths must be %lld contiguous entries", op, (long long)B); return CDR_ERR_BAD_ARG; }
    if (B && !n.data) { set_error("%s: lengths is a null pointer", op); return CDR_ERR_BAD_ARG; }
    if (B && (reinterpret_cast<uintptr_t>(n.data) & (dtype_size(n.dtype) - 1))) { set_error("%s: lengths is not aligned to its type", op); return CDR_ERR_MISALIGNED; }
    a->lengths = n.data;
    a->lengths_i64 = n.dtype == CDR_I64;
  }
  constexpr int64_t kMost = 1 << 30;
  if (B > kMost || Hq > kMost || Sq > kMost || Skv > kMost || P > kMost || (Hkv && Hq / Hkv * Sq > kMost)) {
    set_error("%s: extent too large", op);
    return CDR_ERR_UNSUPPORTED;
  }
  *empty = numel(out) == 0;
  if (int rc = check_pointer(q.data, numel(q), op, "q")) return rc;
  if (int rc = check_pointer(k.data, numel(k), op, "k")) return rc;
  if (int rc = check_pointer(v.data, numel(v), op, "v")) return rc;
  if (int rc = check_pointer(out.data, numel(out), op, "the output")) return rc;
  a->q = q.data; a->k = k.data; a->v = v.data; a->out = out.data;
  a->B = static_cast<int>(B); a->Hq = static_cast<int>(Hq); a->Hkv = static_cast<int>(Hkv);
  a->G = Hkv ? static_cast<int>(Hq / Hkv) : 0;
  a->Sq = static_cast<int>(Sq); a->Skv = static_cast<int>(Skv); a->P = static_cast<int>(P); a->D = static_cast<int>(D);
  a->window = a->sinks = 0;
  a->scale_log2 = scale * 1.4426950408889634f;
  a->bf16 = q.dtype == CDR_BF16;
  return CDR_OK;
}

constexpr int64_t kNoWindow = 1 << 30;   // wider than any cache

int parse_window(const cdr_tensor* ins, int n_in, const cdr_tensor* outs, int n_out, const cdr_window_attn_params* p, CacheAttn* a,
                 bool* empty) {
  if (!p) { set_error("window_attention: params is null"); return CDR_ERR_BAD_ARG; }
  if (p->window < 1 || p->sinks < 0) { set_error("window_attention: window must be at least 1 and sinks at least 0"); return CDR_ERR_BAD_ARG; }
  if (int rc = parse_problem("window_attention", ins, n_in, outs, n_out, false, p->has_lengths, p->scale, a, empty)) return rc;
  a->window = static_cast<int>(p->window < kNoWindow ? p->window : kNoWindow);
  a->sinks = static_cast<int>(p->sinks < kNoWindow ? p->sinks : kNoWindow);
  return CDR_OK;
}

int parse_prefix(const cdr_tensor* ins, int n_in, const cdr_tensor* outs, int n_out, const cdr_prefix_attn_params* p, CacheAttn* a,
                 bool* empty) {
  if (!p) { set_error("prefix_attention: params is null"); return CDR_ERR_BAD_ARG; }
  if (int rc = parse_problem("prefix_attention", ins, n_in, outs, n_out, true, p->has_lengths, p->scale, a, empty)) return rc;
  a->window = kNoWindow;
  return CDR_OK;
}

// Which kernels a call runs.
enum class Path { kStream, kTile, kPacked };

Path choose_path(const CacheAttn& a) {
  if (a.Sq >= 64) return Path::kTile;
  const int64_t rows = static_cast<int64_t>(a.G) * a.Sq;
  if (a.P >= 128 && rows <= 128 && a.B * rows > 32) return Path::kPacked;
  return Path::kStream;
}

size_t cache_attention_workspace(const CacheAttn& a) {
  switch (choose_path(a)) {
    case Path::kTile: return kTileCounterBytes;
    case Path::kPacked: return packed_workspace(a);
    default: return 0;
  }
}

int run_cache_attention(const CacheAttn& a, const char* op, void* ws, size_t ws_bytes, cudaStream_t stream) {
  const Path path = choose_path(a);
  const size_t need = cache_attention_workspace(a);
  if (need && (!ws || ws_bytes < need)) {
    set_error("%s: workspace of %zu bytes required, got %zu", op, need, ws ? ws_bytes : (size_t)0);
    return CDR_ERR_WORKSPACE;
  }
  if (need && !aligned16(ws)) { set_error("%s: workspace must be 16-byte aligned", op); return CDR_ERR_MISALIGNED; }
  PrefixPartials part{nullptr, nullptr, 0, 0};
  if (path == Path::kTile) return launch_tile_attention(a, ws, stream);
  if (path == Path::kPacked)
    if (int rc = launch_packed_prefix(a, ws, &part, stream)) return rc;
  return launch_stream_attention(a, part, stream);
}

}  // namespace

int window_attention_workspace(const cdr_tensor* ins, int n_in, const cdr_tensor* outs, int n_out, const cdr_window_attn_params* p,
                               size_t* bytes) {
  CacheAttn a;
  bool empty = false;
  *bytes = 0;
  if (int rc = parse_window(ins, n_in, outs, n_out, p, &a, &empty)) return rc;
  if (!empty) *bytes = cache_attention_workspace(a);
  return CDR_OK;
}

int prefix_attention_workspace(const cdr_tensor* ins, int n_in, const cdr_tensor* outs, int n_out, const cdr_prefix_attn_params* p,
                               size_t* bytes) {
  CacheAttn a;
  bool empty = false;
  *bytes = 0;
  if (int rc = parse_prefix(ins, n_in, outs, n_out, p, &a, &empty)) return rc;
  if (!empty) *bytes = cache_attention_workspace(a);
  return CDR_OK;
}

int launch_window_attention(const cdr_tensor* ins, int n_in, const cdr_tensor* outs, int n_out, const cdr_window_attn_params* p,
                            void* ws, size_t ws_bytes, cudaStream_t stream) {
  CacheAttn a;
  bool empty = false;
  if (int rc = parse_window(ins, n_in, outs, n_out, p, &a, &empty)) return rc;
  return empty ? CDR_OK : run_cache_attention(a, "window_attention", ws, ws_bytes, stream);
}

int launch_prefix_attention(const cdr_tensor* ins, int n_in, const cdr_tensor* outs, int n_out, const cdr_prefix_attn_params* p,
                            void* ws, size_t ws_bytes, cudaStream_t stream) {
  CacheAttn a;
  bool empty = false;
  if (int rc = parse_prefix(ins, n_in, outs, n_out, p, &a, &empty)) return rc;
  return empty ? CDR_OK : run_cache_attention(a, "prefix_attention", ws, ws_bytes, stream);
}

}  // namespace cdr
