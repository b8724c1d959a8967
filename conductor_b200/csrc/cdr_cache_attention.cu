// K7 -- attention over a key/value cache for few query rows (decode and verification steps):
//   O = softmax(scale * Q K^T [window + sinks, cache length]) V
// for the G * Sq query rows that share one key head of one sequence, and the entry points of
// CDR_T_WINDOW_ATTENTION and CDR_T_PREFIX_ATTENTION.  The reference has no attention over a cache;
// its kernels (choreo-op/attention-gcu-only-test.co:15-134) take q, k and v of one length.
//
// HBM bound: every visible key and value is read once for the (at most 16) rows of a task, a task being
// (sequence, key head, 16-row tile).  The work of all tasks is one list of units of 32 keys, cut into equal
// contiguous shares, one per warp of a grid that is resident as a whole: whatever the lengths, all warps
// finish together.  Each warp runs the online-softmax recurrence on its own, without a barrier:
//   - the TMA unit brings K and V of a unit into the warp's own two-stage ring (16 KB per stage at HD = 128,
//     192 KB in flight per SM); copying them with per-thread 16-byte asynchronous copies instead was
//     bound by instructions and shared-memory traffic (64 sequences below: 126 us, 3.7 TB/s).
//   - the 16-byte pieces are operand registers of m16n8k16 matrix instructions as they are: the order of the
//     contraction index is free as long as both operands use the same one, so a lane takes a piece of a K
//     row (and of the Q row) for two k-steps; for P V it takes a piece of four V rows and pairs them with byte
//     permutes.  With the 128-byte swizzle, lanes c = 0..3 reading pieces 2c + j of a K row, and eight lanes a
//     whole V row, meet no bank conflict.  16 rows are the instruction's height: a task with fewer rows
//     pays nothing for it, the loads set the pace.
//   - the accumulator is rescaled only when a row's maximum grew by more than 2^8; exact after the
//     final division because the sums use the same reference.
// A warp that has all units of a task writes the output, otherwise (maximum, sum, O) in fp32 to scratch; a
// second kernel, launched to overlap this one's tail, adds up each row's parts in a fixed order (no atomics:
// the same call gives the same bits) and those of the shared prefix (cdr_tile_attention.cu).  Where there are
// few tasks, a task belongs to one thread-block cluster instead, whose warps join their parts through
// distributed shared memory: one launch, no scratch (one sequence: 11.2 -> 8.7 us).
// P is rounded to the input type for the second product (WeightShift in cdr_cache_attention.cuh says how far); scores, maxima,
// sums and O stay in fp32.
// Measured (B200): 64 sequences of up to 4096 keys, 32 / 8 heads, window 2048: 85 us, 5.5 TB/s of 465 MB with both
// kernels; long caches (64 x 4096 keys, 2 x 131072) 6.2 TB/s, of 6.5 that a plain copy reaches.  Shorter calls are
// bound by the latency of two dependent launches or of the cluster's exchange.
#include <cuda.h>
#include <math.h>

#include "cdr_cache_attention.cuh"
#include "cdr_sm100.cuh"

namespace cdr {

int make_tensor_map_4d(CUtensorMap* map, const void* base, int is_bf16, const int64_t* dims, const int64_t* strides,
                       const int* box, int swizzle_bytes);

namespace {

constexpr int SA_ROWS = 16;          // query rows of a task (m of the matrix instruction)
constexpr int SA_KEYS = 32;          // keys per unit
constexpr int SA_GROUPS = 2048;      // entries of the table of cumulated units
constexpr float SA_RESCALE = 8.0f;   // log2 units

int make_map(CUtensorMap* m, const void* base, const CacheAttn& a, int64_t S, int64_t H, int64_t B, const HeadStrides& st) {
  const int64_t dims[4] = {a.D, S, H, B}, strides[3] = {st.s, st.h, st.b};
  const int box[4] = {64, SA_KEYS, 1, 1};
  return make_tensor_map_4d(m, base, a.bf16, dims, strides, box, 128);
}

struct StreamArgs {
  CUtensorMap tmap_k, tmap_v, tmap_pk, tmap_pv;   // [B, H, S, D] and the prefix as one sequence; box 64 x 32 keys
  CacheAttn a;
  int* status;
  PrefixPartials part;     // splits > 0: the prefix is already done
  float *slot_o, *slot_ml; // parts: [slot][row of the task][D] and [..][2] = (maximum, sum)
  int* cum;                // [groups + 1] cumulated units, left for the second kernel (lengths given)
  int n_warps;             // shares
  int cluster;             // CTAs per task (CLUSTER)
  int m_tiles;             // tasks per (sequence, key head)
  int group, groups;       // sequences per table entry, table entries
  int rows_cap;            // rows of a slot: min(16, G * Sq)
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

__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr) : "memory");
  return r;
}

// The keys a task reads, as up to three ranges of units of 32 (SA_KEYS): prefix, sinks, window.
struct KeyRanges {
  int prefix_end, sink_end, lo, hi;
  int n_prefix, n_sink, n_total;   // units, cumulated
  bool one_position;               // the live rows see exactly the keys of the ranges
};

__host__ __device__ __forceinline__ int min_(int a, int b) { return a < b ? a : b; }
__host__ __device__ __forceinline__ int max_(int a, int b) { return a > b ? a : b; }

__host__ __device__ __forceinline__ KeyRanges key_ranges(const CacheAttn& a, int prefix, int len, int mt) {
  KeyRanges kr;
  kr.prefix_end = kr.sink_end = kr.lo = kr.hi = 0;
  const int off = len - a.Sq;
  const int r_first = mt * SA_ROWS, r_last = min_(r_first + SA_ROWS, a.G * a.Sq) - 1;   // row r = i * G + g
  const int p_last = off + r_last / a.G, p_first = max_(off + r_first / a.G, 0);        // first row that sees keys
  if (p_last >= 0) {
    kr.prefix_end = prefix;
    kr.hi = p_last + 1;
    kr.lo = max_(p_first - a.window + 1, 0);
    kr.sink_end = min_(a.sinks, kr.lo);
  }
  kr.one_position = p_first == p_last;
  kr.n_prefix = (kr.prefix_end + SA_KEYS - 1) / SA_KEYS;
  kr.n_sink = kr.n_prefix + (kr.sink_end + SA_KEYS - 1) / SA_KEYS;
  kr.n_total = kr.n_sink + (kr.hi - kr.lo + SA_KEYS - 1) / SA_KEYS;
  return kr;
}

// units of one key head of a sequence
__host__ __device__ __forceinline__ int head_units(const CacheAttn& a, int prefix, int len, int m_tiles) {
  int n = 0;
  for (int mt = 0; mt < m_tiles; ++mt) n += key_ranges(a, prefix, len, mt).n_total;
  return n;
}

struct Task {
  int b, hkv, mt, len;
  int first, units;      // its first unit in the list, and how many it has
  KeyRanges kr;
};

// The task that unit u of the list belongs to.
__device__ __forceinline__ Task find_task(const StreamArgs& s, const int* cum, int uniform, int u) {
  const CacheAttn& a = s.a;
  const int prefix = s.part.splits == 0 ? a.P : 0;
  Task t;
  int rest, per_head;
  if (uniform) {                       // no lengths: every sequence has the same units
    per_head = uniform;
    t.b = u / (uniform * a.Hkv);
    rest = u - t.b * (uniform * a.Hkv);
    t.len = a.Skv;
  } else {
    int lo = 0, hi = s.groups - 1;     // last entry with cum <= u
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum[mid] <= u) lo = mid; else hi = mid - 1;
    }
    t.b = lo * s.group;
    rest = u - cum[lo];
    for (;;) {
      t.len = sequence_length(a, t.b);
      per_head = head_units(a, prefix, t.len, s.m_tiles);
      if (rest < per_head * a.Hkv) break;
      rest -= per_head * a.Hkv;
      ++t.b;
    }
  }
  t.hkv = rest / per_head;
  rest -= t.hkv * per_head;
  for (t.mt = 0;; ++t.mt) {
    t.kr = key_ranges(a, prefix, t.len, t.mt);
    if (rest < t.kr.n_total) break;
    rest -= t.kr.n_total;
  }
  t.first = u - rest;
  t.units = t.kr.n_total;
  return t;
}

// Equal shares of the list: share w starts at begin(w); unit u is in share of(u).
struct Shares {
  int n, per, more;      // the first `more` shares have per + 1 units
  __device__ __forceinline__ Shares(int total, int warps) {
    n = min(warps, max(total, 1));     // no share in between is empty
    per = total / n;
    more = total - per * n;
  }
  __device__ __forceinline__ int begin(int w) const { return w * per + min(w, more); }
  __device__ __forceinline__ int of(int u) const {
    const int split = more * (per + 1);
    return u < split ? u / (per + 1) : more + (u - split) / per;
  }
};

// The list of units: cum[e] = units in front of table entry e (lengths given); returns their total, and the units
// of a key head where every sequence has the same.  All THREADS threads of the block take part.
template <int THREADS>
__device__ __forceinline__ int cumulate_units(const StreamArgs& s, int* cum, int* warp_sum, int* uniform) {
  const CacheAttn& a = s.a;
  const int prefix = s.part.splits == 0 ? a.P : 0;
  *uniform = 0;
  if (!a.lengths) {
    *uniform = head_units(a, prefix, a.Skv, s.m_tiles);
    return *uniform * a.Hkv * a.B;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int carry = 0;
  for (int e0 = 0; e0 < s.groups; e0 += THREADS) {
    const int e = e0 + static_cast<int>(threadIdx.x);
    int n = 0;
    if (e < s.groups)
      for (int b = e * s.group; b < min(a.B, (e + 1) * s.group); ++b)
        n += head_units(a, prefix, sequence_length(a, b), s.m_tiles) * a.Hkv;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) x += warp_sum[w];
      all += warp_sum[w];
    }
    if (e < s.groups) cum[e] = carry + x - n;
    carry += all;
    __syncthreads();
  }
  return carry;
}

// 8 columns of an output row as a sum of parts: each part is (maximum, sum of weights, O) in its own reference.
struct RowSum {
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sum = 0.0f, top = -INFINITY;

  __device__ __forceinline__ void join(float m, float l, float4 u, float4 v) {
    const bool none = m == -INFINITY && l == 0.0f; // a part that saw nothing may hold anything; NaN weights stay
    const float m_new = fmaxf(top, m);
    const float f0 = top == -INFINITY ? 0.0f : ex2(top - m_new), f1 = none ? 0.0f : ex2(m - m_new);
    if (none) { l = 0.0f; u = v = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    top = m_new;
    sum = f0 * sum + f1 * l;
    acc[0] = f0 * acc[0] + f1 * u.x; acc[1] = f0 * acc[1] + f1 * u.y; acc[2] = f0 * acc[2] + f1 * u.z; acc[3] = f0 * acc[3] + f1 * u.w;
    acc[4] = f0 * acc[4] + f1 * v.x; acc[5] = f0 * acc[5] + f1 * v.y; acc[6] = f0 * acc[6] + f1 * v.z; acc[7] = f0 * acc[7] + f1 * v.w;
  }
  // parts first, first + step, ... < n; get(i, &o) returns (maximum, sum) of part i and where its 8 columns are.  Four
  // parts are fetched before the first of them is used.
  template <typename Get>
  __device__ __forceinline__ void join_parts(int first, int step, int n, Get get) {
    for (int i0 = first; i0 < n; i0 += 4 * step) {
      float2 ml[4];
      float4 u[4], v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + k * step;
        const float* o;
        ml[k] = get(i < n ? i : i0, &o);
        u[k] = reinterpret_cast<const float4*>(o)[0];
        v[k] = reinterpret_cast<const float4*>(o)[1];
        if (i >= n) ml[k] = make_float2(-INFINITY, 0.0f);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) join(ml[k].x, ml[k].y, u[k], v[k]);
    }
  }
  // with the lane whose number differs in bit x (every lane of the warp calls this)
  __device__ __forceinline__ void join_lane(int x) {
    const float m = __shfl_xor_sync(0xffffffffu, top, x), l = __shfl_xor_sync(0xffffffffu, sum, x);
    float4 u, v;
    u.x = __shfl_xor_sync(0xffffffffu, acc[0], x); u.y = __shfl_xor_sync(0xffffffffu, acc[1], x);
    u.z = __shfl_xor_sync(0xffffffffu, acc[2], x); u.w = __shfl_xor_sync(0xffffffffu, acc[3], x);
    v.x = __shfl_xor_sync(0xffffffffu, acc[4], x); v.y = __shfl_xor_sync(0xffffffffu, acc[5], x);
    v.z = __shfl_xor_sync(0xffffffffu, acc[6], x); v.w = __shfl_xor_sync(0xffffffffu, acc[7], x);
    join(m, l, u, v);
  }
  template <bool BF16>
  __device__ __forceinline__ void store(const CacheAttn& a, int b, int hq, int i, int d) const {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;           // no visible key: 0; NaN passes through
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack16<BF16>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    const int64_t e0 = b * a.so.b + hq * a.so.h + static_cast<int64_t>(i) * a.so.s + d;
    *reinterpret_cast<uint4*>(static_cast<unsigned char*>(a.out) + e0 * 2) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// part n of the shared prefix for one row and 8 of its columns
struct PrefixGet {
  const PrefixPartials& part;
  int64_t row;             // of split 0
  int kv_heads, dim, column;
  __device__ __forceinline__ float2 operator()(int n, const float** o) const {
    const int64_t e = static_cast<int64_t>(n) * kv_heads * part.rows + row;
    *o = part.o + e * dim + column;
    const float lse = part.lse[e];
    return make_float2(lse, lse == -INFINITY ? 0.0f : 1.0f);
  }
};

// what a staged unit is (written with its copies, read when it is used)
struct __align__(16) UnitHeader {
  int base, end;         // first key; one past the last key that may be used
  int flags;             // 1: masked by position  2: starts a segment  4: ends one  8: its task lies in this share as a whole
  int b, hkv, mt, off, task_first;
};

// 192 KB in flight per SM either way; at HD = 64 a unit has half the bytes and about as many dependent steps (8 warps of
// three units: 5.6 against 5.8 TB/s).
template <int HD>
struct StreamSmem {
  static constexpr int WARPS = HD == 128 ? 6 : 12;
  static constexpr int STAGES = 2;                                        // units in flight per warp
  static constexpr int THREADS = WARPS * 32;
  static constexpr int HALF_BYTES = SA_KEYS * HD * 2;          // K or V of a unit
  static constexpr int STAGE_BYTES = 2 * HALF_BYTES;
  static constexpr int HEAD_OFF = WARPS * STAGES * STAGE_BYTES;
  static constexpr int BAR_OFF = HEAD_OFF + WARPS * STAGES * static_cast<int>(sizeof(UnitHeader));
  static constexpr int CUM_OFF = BAR_OFF + WARPS * STAGES * 8;
  static constexpr int FIXED = CUM_OFF + 1024;                 // alignment slack
};

// CLUSTER = false: the list in equal shares, parts to scratch.  CLUSTER = true (few tasks): a task belongs to the warps of
// one thread-block cluster, which add up their parts through distributed shared memory and write the output.
template <int HD, bool BF16, bool CLUSTER>
__global__ void __launch_bounds__(StreamSmem<HD>::THREADS, 1) stream_attention_kernel(const __grid_constant__ StreamArgs args) {
  using L = StreamSmem<HD>;
  constexpr int AC = HD / 64;      // 64-column atoms of a row: 128 bytes, 8 pieces
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* cum = reinterpret_cast<int*>(smem + L::CUM_OFF);
  __shared__ int warp_sum[L::WARPS];
  const CacheAttn& a = args.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  UnitHeader* heads = reinterpret_cast<UnitHeader*>(smem + L::HEAD_OFF) + warp * L::STAGES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF) + warp * L::STAGES;
  unsigned char* ring = smem + warp * (L::STAGES * L::STAGE_BYTES);
  if (lane == 0) {
    if (a.Skv > 0) { sm100::prefetch_tensormap(&args.tmap_k); sm100::prefetch_tensormap(&args.tmap_v); }
    for (int st = 0; st < L::STAGES; ++st) sm100::mbar_init(&bars[st], 1);
    sm100::fence_barrier_init();
  }
  __syncwarp();

  // Behind the packed prefix product this kernel needs nothing of that one, only what came before it, and that one
  // lets its dependents start after its own wait: the wait for it is at the end, for the kernel that adds up.
  const bool behind_prefix = args.part.splits > 0;
  if (!behind_prefix) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");

  int uniform = 0, total, share, n_warps = args.n_warps;
  const int cs = args.cluster, rank = CLUSTER ? static_cast<int>(blockIdx.x) % cs : 0;
  Task lt;
  if constexpr (CLUSTER) {
    const int task = blockIdx.x / cs;                    // the list is this task's alone
    lt.mt = task % args.m_tiles;
    lt.hkv = task / args.m_tiles % a.Hkv;
    lt.b = task / args.m_tiles / a.Hkv;
    lt.len = sequence_length(a, lt.b);
    lt.kr = key_ranges(a, behind_prefix ? 0 : a.P, lt.len, lt.mt);
    lt.first = 0;
    lt.units = total = lt.kr.n_total;
    n_warps = cs * L::WARPS;
    share = warp * cs + rank;
  } else {
    total = cumulate_units<L::THREADS>(args, cum, warp_sum, &uniform);
    if (a.lengths && blockIdx.x == 0)
      for (int e = threadIdx.x; e <= args.groups; e += L::THREADS) args.cum[e] = e < args.groups ? cum[e] : total;
    share = warp * gridDim.x + blockIdx.x;               // neighbouring shares on different SMs
  }
  const Shares shares(total, n_warps);
  const int u_begin = share < shares.n ? shares.begin(share) : 0;
  const int u_end = share < shares.n ? shares.begin(share + 1) : 0;

  // ---- loads run ahead of their use: unit `lu`, in the segment of its task that ends at unit `seg_end`
  int lu = u_begin, seg_end = u_begin;
  auto load_unit = [&](int st) {
    if (lu >= u_end) return;
    const bool starts = lu == seg_end;
    if (starts) {
      if (!CLUSTER) lt = find_task(args, cum, uniform, lu);
      seg_end = min(lt.first + lt.units, u_end);
    }
    if (lane == 0) {
      const int t = lu - lt.first;
      int base, end;
      const bool own = t >= lt.kr.n_prefix;
      if (!own) {
        base = t * SA_KEYS;
        end = lt.kr.prefix_end;
      } else if (t < lt.kr.n_sink) {
        base = (t - lt.kr.n_prefix) * SA_KEYS;
        end = lt.kr.sink_end;
      } else {
        base = lt.kr.lo + (t - lt.kr.n_sink) * SA_KEYS;
        end = lt.kr.hi;
      }
      const void *tk = own ? &args.tmap_k : &args.tmap_pk, *tv = own ? &args.tmap_v : &args.tmap_pv;
      unsigned char* dst = ring + st * L::STAGE_BYTES;
      sm100::mbar_arrive_expect_tx(&bars[st], L::STAGE_BYTES);
#pragma unroll
      for (int j = 0; j < AC; ++j) sm100::tma_load_4d(dst + j * (SA_KEYS * 128), tk, j * 64, base, lt.hkv, own ? lt.b : 0, &bars[st]);
#pragma unroll
      for (int j = 0; j < AC; ++j)
        sm100::tma_load_4d(dst + L::HALF_BYTES + j * (SA_KEYS * 128), tv, j * 64, base, lt.hkv, own ? lt.b : 0, &bars[st]);
      heads[st] = UnitHeader{base, end,
                             (own && !lt.kr.one_position ? 1 : 0) | (starts ? 2 : 0) | (lu + 1 == seg_end ? 4 : 0) |
                                 (lt.first >= u_begin && lt.first + lt.units <= u_end ? 8 : 0),
                             lt.b, lt.hkv, lt.mt, lt.len - a.Sq, lt.first};
    }
    ++lu;
  };
#pragma unroll
  for (int st = 0; st < L::STAGES; ++st) load_unit(st);
  __syncwarp();

  uint4 qf[2][AC][2];
  float o[AC][8][4];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  int pos[2];
  int st = 0, phase = 0;
  for (int u = u_begin; u < u_end; ++u) {
    const UnitHeader h = heads[st];
    const uint32_t kbase = sm100::smem_u32(ring + st * L::STAGE_BYTES), vbase = kbase + L::HALF_BYTES;
    if (h.flags & 2) {
      const int rows = a.G * a.Sq;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = h.mt * SA_ROWS + g + 8 * x;
        const int i = r / a.G, gi = r - i * a.G;
        pos[x] = r < rows ? h.off + i : -1;
        const unsigned char* p = static_cast<const unsigned char*>(a.q) +
                                 (h.b * a.sq.b + static_cast<int64_t>(h.hkv * a.G + gi) * a.sq.h + static_cast<int64_t>(i) * a.sq.s) * 2 + c * 32;
#pragma unroll
        for (int j = 0; j < AC; ++j)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            qf[x][j][y] = r < rows ? __ldg(reinterpret_cast<const uint4*>(p + j * 128 + y * 16)) : make_uint4(0, 0, 0, 0);
        m[x] = -INFINITY;
        l[x] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < AC; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][e][i] = 0.0f;
    }

    if (!__all_sync(0xffffffffu, sm100::mbar_wait(&bars[st], phase))) {       // the whole warp gives up, or none of it
      if (lane == 0) sm100::report_timeout(args.status, 60);
      for (int k = 0; k < L::STAGES && u + k < u_end; ++k)                    // its copies in flight, as long again
        sm100::mbar_wait(&bars[(st + k) % L::STAGES], phase ^ ((st + k) / L::STAGES));
      break;
    }
    float s[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
#pragma unroll
    for (int j = 0; j < AC; ++j)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint4 kf = ld_shared16(kbase + j * (SA_KEYS * 128) + (n * 8 + g) * 128 + (((2 * c + y) ^ g) << 4));
          mma16816<BF16>(s[n], qf[0][j][y].x, qf[1][j][y].x, qf[0][j][y].y, qf[1][j][y].y, kf.x, kf.y);
          mma16816<BF16>(s[n], qf[0][j][y].z, qf[1][j][y].z, qf[0][j][y].w, qf[1][j][y].w, kf.z, kf.w);
        }

    // s[n][2x + e] belongs to row g + 8x and key base + 8n + 2c + e
    const bool own = h.flags & 1, partial = h.base + SA_KEYS > h.end;
    if (own || partial) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = h.base + 8 * n + 2 * c + (i & 1), p = pos[i >> 1];
          if (key >= h.end || (own && (key > p || (key <= p - a.window && key >= a.sinks)))) s[n][i] = -INFINITY;
        }
    }
    float mx[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float v = fmaxf(fmaxf(fmaxf(s[0][2 * x], s[0][2 * x + 1]), fmaxf(s[1][2 * x], s[1][2 * x + 1])),
                      fmaxf(fmaxf(s[2][2 * x], s[2][2 * x + 1]), fmaxf(s[3][2 * x], s[3][2 * x + 1])));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
      // scale > 0: the maximum commutes with it
      mx[x] = fmaf(fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2)), a.scale_log2, -WeightShift<BF16>::value);
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] + SA_RESCALE || mx[1] > m[1] + SA_RESCALE)) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float m_new = fmaxf(m[x], mx[x]);
        const float f = m[x] == -INFINITY ? 0.0f : ex2(m[x] - m_new);
        m[x] = m_new;
        l[x] *= f;
#pragma unroll
        for (int j = 0; j < AC; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) { o[j][e][2 * x] *= f; o[j][e][2 * x + 1] *= f; }
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float ref = m[x] == -INFINITY ? 0.0f : m[x];     // nothing seen yet: every weight is exp2(-inf) = 0
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = ex2(fmaf(s[n][2 * x + e], a.scale_log2, -ref));
          s[n][2 * x + e] = p;
          l[x] += p;
        }
    }
#pragma unroll
    for (int kk = 0; kk < SA_KEYS / 16; ++kk) {
      const uint32_t pa0 = pack16<BF16>(s[2 * kk][0], s[2 * kk][1]), pa1 = pack16<BF16>(s[2 * kk][2], s[2 * kk][3]);
      const uint32_t pa2 = pack16<BF16>(s[2 * kk + 1][0], s[2 * kk + 1][1]), pa3 = pack16<BF16>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
      for (int j = 0; j < AC; ++j) {
        uint4 vf[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int row = kk * 16 + (n >> 1) * 8 + 2 * c + (n & 1);
          vf[n] = ld_shared16(vbase + j * (SA_KEYS * 128) + row * 128 + ((g ^ (2 * c + (n & 1))) << 4));
          // a weight of 0 must not meet what the cache holds behind the range
          if (partial && h.base + row >= h.end) vf[n] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t v0 = (&vf[0].x)[w], v1 = (&vf[1].x)[w], v2 = (&vf[2].x)[w], v3 = (&vf[3].x)[w];
          mma16816<BF16>(o[j][2 * w], pa0, pa1, pa2, pa3, __byte_perm(v0, v1, 0x5410), __byte_perm(v2, v3, 0x5410));
          mma16816<BF16>(o[j][2 * w + 1], pa0, pa1, pa2, pa3, __byte_perm(v0, v1, 0x7632), __byte_perm(v2, v3, 0x7632));
        }
      }
    }
    __syncwarp();                                // every lane is done with the stage and its header
    load_unit(st);
    __syncwarp();
    if (++st == L::STAGES) { st = 0; phase ^= 1; }

    if (!CLUSTER && (h.flags & 4)) {
      // ---- end of a segment: o[j][e][2x + i] is row g + 8x, column 64 j + 8 (2c + i) + e
      const int rows = min(SA_ROWS, a.G * a.Sq - h.mt * SA_ROWS);
      const bool whole = h.flags & 8;
      const int task = (h.b * a.Hkv + h.hkv) * args.m_tiles + h.mt;
      const int64_t slot = whole ? 2LL * args.n_warps + task : 2LL * share + (h.task_first <= u_begin ? 0 : 1);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        const int row = g + 8 * x;
        if (row >= rows) continue;
        if (whole && !behind_prefix) {
          const int r = h.mt * SA_ROWS + row, i = r / a.G, gi = r - i * a.G;
          const float inv = l[x] == 0.0f ? 0.0f : 1.0f / l[x];       // no visible key: 0; NaN passes through
          const bool sees = pos[x] >= 0;
          unsigned char* p = static_cast<unsigned char*>(a.out) +
                             (h.b * a.so.b + static_cast<int64_t>(h.hkv * a.G + gi) * a.so.h + static_cast<int64_t>(i) * a.so.s) * 2 + c * 32;
#pragma unroll
          for (int j = 0; j < AC; ++j)
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = sees ? pack16<BF16>(o[j][2 * e][2 * x + i2] * inv, o[j][2 * e + 1][2 * x + i2] * inv) : 0u;
              *reinterpret_cast<uint4*>(p + j * 128 + i2 * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
          const int64_t at = slot * args.rows_cap + row;
          if (c == 0) *reinterpret_cast<float2*>(args.slot_ml + at * 2) = make_float2(m[x], l[x]);
          float* p = args.slot_o + at * HD + c * 16;
#pragma unroll
          for (int j = 0; j < AC; ++j)
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2)
#pragma unroll
              for (int e = 0; e < 8; e += 4)
                *reinterpret_cast<float4*>(p + j * 64 + i2 * 8 + e) =
                    make_float4(o[j][e][2 * x + i2], o[j][e + 1][2 * x + i2], o[j][e + 2][2 * x + i2], o[j][e + 3][2 * x + i2]);
        }
      }
    }
  }
  if (behind_prefix) asm volatile("griddepcontrol.wait;" ::: "memory");
  if constexpr (CLUSTER) {
    // ---- every warp's part in its ring (all its units are used), then the live rows' 8-column pieces are shared out over
    // the CTAs; `tpp` neighbouring threads take the parts of a piece (the cluster's warps, then the prefix's) in turn
    constexpr int PITCH = HD + 4, VECS = HD / 8;
    __shared__ float2 sm_ml[L::WARPS][SA_ROWS];
    float* part = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      const int row = g + 8 * x;
      if (c == 0) sm_ml[warp][row] = make_float2(m[x], l[x]);
      if (u_begin < u_end) {
#pragma unroll
        for (int j = 0; j < AC; ++j)
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2)
#pragma unroll
            for (int e = 0; e < 8; e += 4)
              *reinterpret_cast<float4*>(part + row * PITCH + c * 16 + j * 64 + i2 * 8 + e) =
                  make_float4(o[j][e][2 * x + i2], o[j][e + 1][2 * x + i2], o[j][e + 2][2 * x + i2], o[j][e + 3][2 * x + i2]);
      }
    }
    if (cs > 1) sm100::cluster_sync_all(); else __syncthreads();
    const int rows = a.G * a.Sq, r_first = lt.mt * SA_ROWS, r_live = min(SA_ROWS, rows - r_first);
    const int pieces = r_live * VECS, per_cta = (pieces + cs - 1) / cs, n_parts = cs * L::WARPS;
    int tpp = 1;
    while (tpp < 16 && tpp * 2 * per_cta <= L::THREADS) tpp *= 2;
    const int sub = threadIdx.x % tpp;
    const int at_once = L::THREADS / tpp, passes = (per_cta + at_once - 1) / at_once;
    for (int pass = 0; pass < passes; ++pass) {
      const int w = pass * at_once + static_cast<int>(threadIdx.x) / tpp;
      const int piece = rank * per_cta + w;
      const bool live = w < per_cta && piece < pieces;
      const int row = live ? piece / VECS : 0, d = live ? piece % VECS * 8 : 0;
      const int r = r_first + row, i = r / a.G, gi = r - i * a.G;
      RowSum sum;
      if (live && lt.len - a.Sq + i >= 0) {
        sum.join_parts(sub, tpp, n_parts, [&](int n, const float** o) {
          const int wn = n % L::WARPS, cn = n / L::WARPS;
          const float2* pml = &sm_ml[wn][row];
          *o = reinterpret_cast<const float*>(smem + wn * (L::STAGES * L::STAGE_BYTES)) + row * PITCH + d;
          if (cs > 1) {
            pml = static_cast<const float2*>(__cluster_map_shared_rank(pml, cn));
            *o = static_cast<const float*>(__cluster_map_shared_rank(*o, cn));
          }
          return *pml;
        });
        if (behind_prefix) sum.join_parts(sub, tpp, args.part.splits, PrefixGet{args.part, args.part.row_of(a, lt.b, i, gi) + static_cast<int64_t>(lt.hkv) * args.part.rows, a.Hkv, HD, d});
      }
      for (int x = 1; x < tpp; x *= 2) sum.join_lane(x);
      if (live && sub == 0) sum.template store<BF16>(a, lt.b, lt.hkv * a.G + gi, i, d);
    }
    if (cs > 1) sm100::cluster_sync_all();       // no CTA leaves while another still reads its parts
  }
}

// Adds up the parts of every row that no warp finished alone: `tpr` threads per row, 8 columns each, which take
// the row's parts in turn (in the order of the keys, then the prefix's).
constexpr int CA_THREADS = 256;

template <int HD, bool BF16>
__global__ void __launch_bounds__(CA_THREADS) combine_parts_kernel(const __grid_constant__ StreamArgs args, int tpr) {
  constexpr int VECS = HD / 8;
  __shared__ float sm_acc[CA_THREADS / 32][VECS][8], sm_ms[CA_THREADS / 32][VECS][2];
  const CacheAttn& a = args.a;
  const int prefix = args.part.splits == 0 ? a.P : 0;
  const int rows = a.G * a.Sq;
  const int64_t row_all = static_cast<int64_t>(blockIdx.x) * (CA_THREADS / tpr) + threadIdx.x / tpr;
  const int64_t n_rows = static_cast<int64_t>(a.B) * a.Hkv * rows;
  const bool live = row_all < n_rows;
  const int r = live ? static_cast<int>(row_all % rows) : 0;
  const int bh = live ? static_cast<int>(row_all / rows) : 0;
  const int hkv = bh % a.Hkv, b = bh / a.Hkv;
  const int i = r / a.G, gi = r - i * a.G;
  const int mt = r / SA_ROWS, row = r - mt * SA_ROWS;
  const int t = threadIdx.x % tpr, vec = t % VECS, sub = t / VECS, nsub = tpr / VECS;

  // the task's units, and the shares that hold them
  const int len = sequence_length(a, b);
  const int per_head = head_units(a, prefix, len, args.m_tiles);
  // (the lengths were there before the first of the kernels started; what that one left is there after the wait)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  int first, total;
  if (!a.lengths) {
    first = per_head * (b * a.Hkv + hkv);
    total = per_head * a.Hkv * a.B;
  } else {
    const int e = b / args.group;
    first = args.cum[e] + per_head * hkv;
    total = args.cum[args.groups];
    for (int x = e * args.group; x < b; ++x) first += head_units(a, prefix, sequence_length(a, x), args.m_tiles) * a.Hkv;
  }
  for (int x = 0; x < mt; ++x) first += key_ranges(a, prefix, len, x).n_total;
  const int units = key_ranges(a, prefix, len, mt).n_total;
  const Shares shares(total, args.n_warps);
  int w0 = 0, w1 = -1, first_slot = 0;
  if (units > 0) {
    w0 = shares.of(first);
    w1 = shares.of(first + units - 1);
    first_slot = first <= shares.begin(w0) ? 0 : 1;        // the later shares start inside the task: their slot 0
  }
  const bool behind_prefix = args.part.splits > 0;
  const bool done = !live || (w0 == w1 && !behind_prefix);       // written by the warp that had it all
  const bool sees = !done && len - a.Sq + i >= 0;
  const int task = (b * a.Hkv + hkv) * args.m_tiles + mt;

  RowSum sum;
  if (sees) {
    sum.join_parts(w0 + sub, nsub, w1 + 1, [&](int w, const float** o) {
      const int64_t slot = w0 == w1 ? 2LL * args.n_warps + task : 2LL * w + (w == w0 ? first_slot : 0);
      const int64_t at = slot * args.rows_cap + row;
      *o = args.slot_o + at * HD + vec * 8;
      return *reinterpret_cast<const float2*>(args.slot_ml + at * 2);
    });
    if (behind_prefix) sum.join_parts(sub, nsub, args.part.splits, PrefixGet{args.part, args.part.row_of(a, b, i, gi) + static_cast<int64_t>(hkv) * args.part.rows, a.Hkv, HD, vec * 8});
  }
  // lanes of a warp with the same columns, then the row's warps
  for (int x = VECS; x < 32; x *= 2) sum.join_lane(x);
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane < VECS) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sm_acc[warp][lane][e] = sum.acc[e];
      sm_ms[warp][lane][0] = sum.top;
      sm_ms[warp][lane][1] = sum.sum;
    }
    __syncthreads();
    if (sub == 0) {
      for (int w = warp + 1; w < warp + tpr / 32; ++w) {
        const float* p = sm_acc[w][vec];
        sum.join(sm_ms[w][vec][0], sm_ms[w][vec][1], make_float4(p[0], p[1], p[2], p[3]), make_float4(p[4], p[5], p[6], p[7]));
      }
    }
  }
  if (!done && sub == 0) sum.template store<BF16>(a, b, hkv * a.G + gi, i, vec * 8);
}

// ---------------------------------------------------------------- host side
// Clusters of 2, 4, 8 CTAs that the current device holds at once (a GPC of 16 or 18 SMs does not always take two of eight).
int max_clusters(int D, int size);

// `packed`: behind the packed prefix product, on the SMs that it leaves
StreamPlan plan_stream(const CacheAttn& a, const PackedPlan* packed) {
  StreamPlan p;
  const int warps = a.D == 128 ? StreamSmem<128>::WARPS : StreamSmem<64>::WARPS;
  const int64_t rows = static_cast<int64_t>(a.G) * a.Sq;
  p.m_tiles = static_cast<int>((rows + SA_ROWS - 1) / SA_ROWS);
  p.rows_cap = static_cast<int>(rows < SA_ROWS ? rows : SA_ROWS);
  p.tasks = static_cast<int64_t>(a.B) * a.Hkv * p.m_tiles;
  const int prefix = packed ? 0 : a.P;
  int64_t per_head = 0;
  for (int mt = 0; mt < p.m_tiles; ++mt) per_head += key_ranges(a, prefix, a.Skv, mt).n_total;
  p.units = per_head * a.B * a.Hkv;
  const int64_t sms = packed ? (sm_count() > packed->ctas ? sm_count() - packed->ctas : 1) : sm_count();
  p.cluster = 0;
  if (p.tasks <= sms) {
    p.cluster = 1;
    while (p.cluster < 8 && p.tasks * p.cluster * 2 <= sms && per_head > p.m_tiles * p.cluster * warps && p.tasks <= max_clusters(a.D, p.cluster * 2))
      p.cluster *= 2;
    // long shares: the list fills all SMs and reads 6 TB/s, clusters of 128 CTAs 4 (2 sequences of 131072 keys: 267 us so)
    if (per_head > 8LL * p.m_tiles * p.cluster * warps) p.cluster = 0;
  }
  // every warp the machine can hold at once, if there is a unit for each
  p.ctas = static_cast<int>(p.units < sms ? (p.units < 1 ? 1 : p.units) : sms);
  p.n_warps = p.ctas * warps;
  p.group = (a.B + SA_GROUPS - 1) / SA_GROUPS;
  p.groups = (a.B + p.group - 1) / p.group;
  p.slots = p.cluster ? 0 : 2LL * p.n_warps + (packed ? p.tasks : 0);
  return p;
}

size_t table_bytes(const StreamPlan& p) { return (static_cast<size_t>(p.groups + 1) * sizeof(int) + 255) / 256 * 256; }

size_t stream_bytes(const CacheAttn& a, const StreamPlan& p) {
  return p.cluster ? 0 : table_bytes(p) + static_cast<size_t>(p.slots) * p.rows_cap * (a.D + 2) * sizeof(float);
}

template <int HD, bool BF16, bool CLUSTER>
cudaError_t configure_stream() {
  constexpr int most = StreamSmem<HD>::FIXED + SA_GROUPS * static_cast<int>(sizeof(int));
  return cudaFuncSetAttribute(stream_attention_kernel<HD, BF16, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
}

template <int HD>
int query_clusters(int size) {
  if (configure_stream<HD, true, true>() != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(size), 1, 1);
  cfg.blockDim = dim3(StreamSmem<HD>::THREADS, 1, 1);
  cfg.dynamicSmemBytes = StreamSmem<HD>::FIXED;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(size);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, stream_attention_kernel<HD, true, true>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return n;
}

int max_clusters(int D, int size) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  static int known[64][2][4] = {};             // count + 1; a race stores the same value twice
  int& k = known[dev][D == 128][size == 2 ? 1 : size == 4 ? 2 : 3];
  if (k == 0) k = 1 + (D == 128 ? query_clusters<128>(size) : query_clusters<64>(size));
  return k - 1;
}

template <int HD, bool BF16>
int launch_stream_cfg(const StreamArgs& s, const StreamPlan& p, int tpr, cudaStream_t stream) {
  using L = StreamSmem<HD>;
  const size_t table = s.a.lengths && !p.cluster ? s.groups * sizeof(int) : 0;
  int dev = 0;
  CDR_CUDA_TRY(cudaGetDevice(&dev));
  static bool configured_dev[64] = {false};
  if (!configured_dev[dev & 63]) {
    CDR_CUDA_TRY((configure_stream<HD, BF16, false>()));
    CDR_CUDA_TRY((configure_stream<HD, BF16, true>()));
    configured_dev[dev & 63] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.blockDim = dim3(L::THREADS, 1, 1);
  cfg.dynamicSmemBytes = L::FIXED + table;
  cfg.stream = stream;
  if (p.cluster) {
    cfg.gridDim = dim3(static_cast<unsigned>(p.tasks * p.cluster), 1, 1);
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(p.cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
    CDR_CUDA_TRY(cudaLaunchKernelEx(&cfg, stream_attention_kernel<HD, BF16, true>, s));
    return CDR_OK;
  }
  cfg.gridDim = dim3(static_cast<unsigned>(p.ctas), 1, 1);
  CDR_CUDA_TRY(cudaLaunchKernelEx(&cfg, stream_attention_kernel<HD, BF16, false>, s));
  const int64_t rows = static_cast<int64_t>(s.a.B) * s.a.Hq * s.a.Sq;
  cfg.gridDim = dim3(static_cast<unsigned>((rows + CA_THREADS / tpr - 1) / (CA_THREADS / tpr)), 1, 1);
  cfg.blockDim = dim3(CA_THREADS, 1, 1);
  cfg.dynamicSmemBytes = 0;
  CDR_CUDA_TRY(cudaLaunchKernelEx(&cfg, combine_parts_kernel<HD, BF16>, s, tpr));
  return CDR_OK;
}

}  // namespace

namespace {

int launch_stream_attention(const CacheAttn& a, const StreamPlan& p, const PrefixPartials& part, void* ws, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq * a.Sq;
  if (p.units > 0x3fffffff || p.tasks > 0x3fffffff || rows > 0x3fffffff) { set_error("attention: too many row tiles for one launch"); return CDR_ERR_UNSUPPORTED; }
  StreamArgs s = {};
  s.a = a;
  s.part = part;
  s.status = device_status_ptr();
  if (a.Skv > 0) {           // an empty cache, or prefix, is never loaded from
    if (int rc = make_map(&s.tmap_k, a.k, a, a.Skv, a.Hkv, a.B, a.sk)) return rc;
    if (int rc = make_map(&s.tmap_v, a.v, a, a.Skv, a.Hkv, a.B, a.sv)) return rc;
  }
  if (a.P > 0 && part.splits == 0) {
    if (int rc = make_map(&s.tmap_pk, a.pk, a, a.P, a.Hkv, 1, a.spk)) return rc;
    if (int rc = make_map(&s.tmap_pv, a.pv, a, a.P, a.Hkv, 1, a.spv)) return rc;
  }
  s.cum = static_cast<int*>(ws);
  s.slot_o = reinterpret_cast<float*>(static_cast<unsigned char*>(ws) + table_bytes(p));
  s.slot_ml = s.slot_o + p.slots * p.rows_cap * a.D;
  s.n_warps = p.n_warps;
  s.cluster = p.cluster;
  s.m_tiles = p.m_tiles;
  s.group = p.group;
  s.groups = p.groups;
  s.rows_cap = p.rows_cap;
  // threads per row of the second kernel, by the parts that a row may have; a CTA per row pays only where there are few
  // rows.  Whole calls with 32 / 64 / 256 threads, us: 32 rows (131072 keys) 113 / 102 / 94, 64 rows (16384 keys) 43 / 37 / 32;
  // 2048 rows behind a prefix of 65536 keys 97 / 94 / 109; 8192 rows behind 32768 keys, few parts, 180 / 192 / 232.
  const int64_t per_task = p.tasks ? p.units / p.tasks : 0, per_warp = p.units / p.n_warps + 1;
  const int64_t parts = per_task / per_warp + 1 + part.splits;
  const int tpr = rows <= 2 * sm_count() && parts > 16 ? 256 : parts <= 8 ? 32 : 64;
  if (a.D == 128) return a.bf16 ? launch_stream_cfg<128, true>(s, p, tpr, stream) : launch_stream_cfg<128, false>(s, p, tpr, stream);
  return a.bf16 ? launch_stream_cfg<64, true>(s, p, tpr, stream) : launch_stream_cfg<64, false>(s, p, tpr, stream);
}

// ---------------------------------------------------------------- entry points

// [.., S, D] operand: D contiguous, every other stride a positive multiple of 16 bytes.  Extents of 1
// get a stride that the kernels may use for address arithmetic.
int check_operand(const cdr_tensor& t, const char* op, const char* name, int rank, int dtype, int64_t D, HeadStrides* st) {
  if (t.rank != rank) { set_error("%s: %s has rank %d, expected %d", op, name, t.rank, rank); return CDR_ERR_BAD_ARG; }
  if (t.dtype != dtype) { set_error("%s: %s differs from q in dtype", op, name); return CDR_ERR_BAD_ARG; }
  if (t.shape[rank - 1] != D) { set_error("%s: %s has head dimension %lld, q has %lld", op, name, (long long)t.shape[rank - 1], (long long)D); return CDR_ERR_BAD_ARG; }
  *st = HeadStrides{D, D, D};
  if (numel(t) == 0) return CDR_OK;      // never addressed: whatever strides a view of nothing has
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
  // (in powers of two too, as the kernels use it: an infinite factor would turn scores of 0 into NaN)
  if (!(scale > 0.0f) || !isfinite(scale * 1.4426950408889634f)) { set_error("%s: scale must be positive and finite", op); return CDR_ERR_UNSUPPORTED; }
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

// Which kernels a call runs, and their scratch.
enum class Path { kStream, kTile, kPacked };

struct CachePlan {
  Path path;
  PackedPlan packed;
  StreamPlan stream;
  size_t packed_bytes, bytes;      // of the product's part of the scratch, of all
};

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// By estimated times in us (B200).  Streaming: 6 per call and, per unit of 32 keys that a warp takes in turn, 1.7 where the rows
// of a task share one position and 2.8 where they do not.  Tiles: 6 and 2.0 per round of 128-key blocks.  Measured:
// 8 sequences, 32 / 8 heads, 4096 keys: 16 queries 97 streamed / 128 in tiles, 24 queries 144 / 128; 1 sequence: 48 queries
// 49 / 63.  Prefix of 4096 keys, 8 heads, 64 own keys: 4 sequences 14 streamed / 18 packed, 8 sequences 24 / 18, 64 118 / 21;
// of 16384: 2 sequences 24 / 29, 4 sequences 37 / 33.
// The streaming estimate has no term for the memory's rate: one sequence of 131072 keys is put at 69 and takes 93.
// From 256 queries on tiles are taken without an estimate, whose walk over all row tiles would cost a prompt's call more than its
// launch.  That is right where the heads fill the machine and wrong where few of them stand before a long cache; 256 queries, us,
// tiles / streamed: 8 sequences of 32 / 8 heads, 4096 keys 141 / 1751; 1 of 32 / 8, 8192 keys 131 / 408, window 512 21 / 112;
// but 1 of 8 / 8, 4096 keys 68 / 61; 1 of 4 / 4, 32768 keys 496 / 184.
CachePlan plan_call(const CacheAttn& a) {
  CachePlan c;
  c.packed_bytes = 0;
  if (a.Sq >= 256) {
    c.path = Path::kTile;
    c.bytes = kTileCounterBytes;
    return c;
  }
  const int warps = sm_count() * (a.D == 128 ? StreamSmem<128>::WARPS : StreamSmem<64>::WARPS);
  const float unit_us = a.Sq == 1 ? 1.7f : 2.8f;
  c.stream = plan_stream(a, nullptr);
  const float stream_us = 6.0f + c.stream.units * unit_us / warps;
  const float tile_us = tile_attention_us(a);
  const int64_t rows = static_cast<int64_t>(a.G) * a.Sq;
  if (a.P >= 128 && rows <= 128 && a.B > 1) {
    const PackedPlan packed = plan_packed(a, c.stream.units - static_cast<int64_t>(c.stream.tasks) * ((a.P + SA_KEYS - 1) / SA_KEYS));
    if (packed.us < stream_us && packed.us < tile_us) {
      c.path = Path::kPacked;
      c.packed = packed;
      c.stream = plan_stream(a, &packed);
      c.packed_bytes = round256(packed_workspace(a, packed));
      c.bytes = c.packed_bytes + stream_bytes(a, c.stream);
      return c;
    }
  }
  // A single query is always streamed: there every row of a task stands at one position, so keys that it does not see are
  // never multiplied, whatever the cache holds there; a tile would meet them at the edges of its blocks with a weight of 0.
  c.path = a.Sq > 1 && tile_us < stream_us ? Path::kTile : Path::kStream;
  c.bytes = c.path == Path::kTile ? kTileCounterBytes : stream_bytes(a, c.stream);
  return c;
}

int run_cache_attention(const CacheAttn& a, const char* op, void* ws, size_t ws_bytes, cudaStream_t stream) {
  const CachePlan c = plan_call(a);
  if (c.bytes && (!ws || ws_bytes < c.bytes)) {
    set_error("%s: workspace of %zu bytes required, got %zu", op, c.bytes, ws ? ws_bytes : (size_t)0);
    return CDR_ERR_WORKSPACE;
  }
  if (c.bytes && (reinterpret_cast<uintptr_t>(ws) & 31u)) { set_error("%s: workspace must be 32-byte aligned", op); return CDR_ERR_MISALIGNED; }
  if (c.path == Path::kTile) return launch_tile_attention(a, ws, stream);
  PrefixPartials part{nullptr, nullptr, 0, 0, 1};
  if (c.path == Path::kPacked) {
    if (int rc = launch_packed_prefix(a, c.packed, ws, &part, stream)) return rc;
    ws = static_cast<unsigned char*>(ws) + c.packed_bytes;
  }
  return launch_stream_attention(a, c.stream, part, ws, stream);
}

}  // namespace

int window_attention_workspace(const cdr_tensor* ins, int n_in, const cdr_tensor* outs, int n_out, const cdr_window_attn_params* p,
                               size_t* bytes) {
  CacheAttn a;
  bool empty = false;
  *bytes = 0;
  if (int rc = parse_window(ins, n_in, outs, n_out, p, &a, &empty)) return rc;
  if (!empty) *bytes = plan_call(a).bytes;
  return CDR_OK;
}

int prefix_attention_workspace(const cdr_tensor* ins, int n_in, const cdr_tensor* outs, int n_out, const cdr_prefix_attn_params* p,
                               size_t* bytes) {
  CacheAttn a;
  bool empty = false;
  *bytes = 0;
  if (int rc = parse_prefix(ins, n_in, outs, n_out, p, &a, &empty)) return rc;
  if (!empty) *bytes = plan_call(a).bytes;
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
