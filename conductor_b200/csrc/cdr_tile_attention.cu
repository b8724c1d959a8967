// K8 -- attention over a key/value cache for many query rows: prompts and chunks of prompts (window and
// prefix attention) and the shared prefix of a batch, whose rows are packed into one matrix product.
//
// Tensor-core bound.  The machine is that of cdr_attention.cu: persistent CTAs, one per SM; a tile is
// 256 query rows in two 128-row halves that share every K/V block of 128 keys and take turns on the tensor
// core; S = Q K^T (tcgen05, fp32 in tensor memory), softmax by one thread per row, P as 16-bit pairs
// over the S columns, O += P V with P read from tensor memory; K and V through one 4-stage TMA ring.
//   warp 0 TMA producer, warp 1 MMA issuer, warps 2-3 idle, warps 4-7 / 8-11 softmax of half A / B
// (register split, barriers, reference-maximum rule: see that file).  What is different:
//   - a tile walks a LIST of key blocks instead of a prefix of them: the shared prefix's blocks, the
//     blocks that hold the sinks, then the blocks that its rows' windows touch.  Each half skips the blocks that
//     none of its rows sees, so a window of W keys costs W / 128 + 2 blocks per half, wherever it lies.
//   - query i stands at position L - Sq + i with L read per sequence by the producer warp, which hands it
//     to the other warps with the tile index.  Masks are applied on the blocks at the edges only.
//   - the cache behind L may hold anything: its scores are masked, and its V rows, which would turn a
//     zero weight into NaN, are cleared in shared memory by the MMA warp (last block of a sequence only).
//   - a first block that holds nothing but up to 32 sinks is cut to 32 keys (two k-steps of P V, 32 columns of softmax):
//     with a window of 512 keys it would else be a sixth of the work (8 x 2048 prompt, 128 -> 122 us).
//   - PACKED (shared prefix): the 128 rows of a half are the G*Sq rows of several sequences that share a key
//     head, fetched by one 4-D box; the prefix is split over tiles and O / l and log2 of the sum go to
//     scratch in fp32, where the streaming kernel joins them with the sequences' own keys.
// What bounds it: the chain softmax -> own products -> softmax of a half, and the MMA warp, which in a build with clocks in
// the kernel was busy for 2950 of the 3770 cycles of a block pair (32 products of 64.6 cycles, see cdr_attention.cu, are
// 2067 of them; the rest are barriers, commits and hand-overs).  Measured
// (B200, twelve calls at a time in a captured graph; a loop of calls under the power limit in brackets): 4 x 1024 queries behind
// 4096 shared keys 166 us [180], 0.93 PFLOP/s [0.86] of 1.60 that a large library product reaches; an 8192 prompt with a
// window of 2048 268 us [293], 0.90 [0.82]; 8 x 2048 with a window of 512 116 us [125], 0.52 [0.48] (masked halves of
// edge blocks, and an epilogue every 5 blocks).
// P is rounded to the input type for the second product, as in cdr_cache_attention.cu.
// Measured and dropped: products cut to the visible keys in every edge block (operand shapes that the issuing warp computes
// at run time: 172 -> 205 us on the first case).
#include <cuda.h>
#include <math.h>

#include "cdr_attention_softmax.cuh"
#include "cdr_cache_attention.cuh"
#include "cdr_common.cuh"
#include "cdr_sm100.cuh"

namespace cdr {

int make_tensor_map_4d(CUtensorMap* map, const void* base, int is_bf16, const int64_t* dims, const int64_t* strides,
                       const int* box, int swizzle_bytes);

namespace {

constexpr int HALF = 128, BQ = 256, BKV = 128;    // rows per half, per tile; keys per block
constexpr int TA_THREADS = 384, SOFTMAX_WARP0 = 4;
constexpr int REGS_CONTROL = 88, REGS_SOFTMAX = 208;   // 128*88 + 256*208 <= 384*168, the CTA's allocation at launch
constexpr int TMEM_S = 0, TMEM_O = 256, TMEM_COLS = 512;   // + 128 * half
constexpr float kRescale = 8.0f;                  // log2 units
constexpr int SINK_COLS = 32;                     // a block of sinks alone is cut to so many keys
constexpr int KV_STAGES = 4, TILE_SLOTS = 4, TILE_READERS = 9;

struct TileArgs {
  CUtensorMap tmap_q, tmap_k, tmap_v, tmap_pk, tmap_pv, tmap_o;
  CacheAttn a;
  unsigned int* next_tile;   // scratch: tiles handed out beyond the first per CTA (nullptr: there are none)
  int* status;
  int n_qtiles, group_heads, total_tiles;
  // PACKED
  int seqs_per_half, split_blocks, splits;
  float *part_o, *part_lse;
  int part_rows;
};

template <int HD>
struct TileSmem {
  static constexpr int TILE_BYTES = 128 * HD * 2;
  static constexpr int Q_OFF = 0;
  static constexpr int KV_OFF = 2 * TILE_BYTES;
  static constexpr int BAR_OFF = KV_OFF + KV_STAGES * TILE_BYTES;
  static constexpr int STAGE_OFF = BAR_OFF + 1024;
  // 8 softmax warps x two stages of 32 rows x 32 16-bit columns (PACKED: one of fp32 columns)
  static constexpr int WARP_STAGE = 2 * 32 * 64;
  static constexpr size_t TOTAL = STAGE_OFF + 8 * WARP_STAGE + 1024;
};

enum { B_QFULL = 0, B_QEMPTY = 1, B_FULL = 2, B_EMPTY = B_FULL + KV_STAGES, B_SFULL = B_EMPTY + KV_STAGES, B_PFULL = B_SFULL + 2,
       B_PVDONE = B_PFULL + 2, B_OFREE = B_PVDONE + 2, B_TFULL = B_OFREE + 2, B_TEMPTY = B_TFULL + TILE_SLOTS,
       B_DRAIN = B_TEMPTY + TILE_SLOTS, B_COUNT };
static_assert(B_COUNT * 8 + 8 + TILE_SLOTS * 8 <= 256, "barrier block");

// One tile: its rows and its list of key blocks.  Entry j of the list is prefix block p0 + j for j < np, else
// the sequence's own block own_block(j).
struct Tile {
  int b, hq, hkv, q0;        // sequence, heads, first query (PACKED: b is the first sequence of half A)
  int off;                   // position of query 0
  int p0, np;                // prefix blocks
  int ns, wstart;            // own blocks: [0, ns) and [wstart, ...)
  int n_iter;
  int live[2];               // the half has rows that see keys
  int pre[2], wa[2], wb[2];  // it takes part in entries [0, pre) and [wa, wb]
  int light[2];              // entry 0 holds nothing but at most 32 sinks for the half

  __device__ __forceinline__ int own_block(int j) const { const int o = j - np; return o < ns ? o : wstart + o - ns; }
  __device__ __forceinline__ bool active(int h, int j) const {   // h: known to the compiler
    return j < pre[h] || (j >= wa[h] && j <= wb[h]);
  }
};

// The first block of a tile when it is sinks alone: `see` of its 32 columns are visible to this row.
template <bool BF16>
__device__ __forceinline__ void softmax_sinks(int see, float scale_log2, uint32_t s_taddr, float& m_ref, float& l) {
  uint32_t sr[SINK_COLS], pw[SINK_COLS / 2];
  sm100::tmem_ld32(s_taddr, sr);
  sm100::tmem_ld_wait();
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < SINK_COLS; ++i) {
    if (i >= see) sr[i] = __float_as_uint(-INFINITY);
    top = fmaxf(top, __uint_as_float(sr[i]));
  }
  m_ref = fmaf(top, scale_log2, -WeightShift<BF16>::value);
  const float neg_m = m_ref == -INFINITY ? 0.0f : -m_ref;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < SINK_COLS; i += 2) {
    const float p0 = fast_exp2(fmaf(__uint_as_float(sr[i]), scale_log2, neg_m)), p1 = fast_exp2(fmaf(__uint_as_float(sr[i + 1]), scale_log2, neg_m));
    sum += p0 + p1;
    pw[i / 2] = pack_pair<BF16>(p0, p1);
  }
  l = sum;
  sm100::tmem_st16(s_taddr, pw);
}

template <bool PACKED>
__device__ __forceinline__ void decode_tile(const TileArgs& t, int idx, int len, Tile& r) {
  const CacheAttn& a = t.a;
  if (PACKED) {
    // row tiles innermost, then heads: the tiles in flight share the prefix's blocks in L2
    const int rt = idx % t.n_qtiles, x = idx / t.n_qtiles;
    r.hkv = x % a.Hkv;
    const int split = x / a.Hkv;
    r.b = rt * 2 * t.seqs_per_half;
    r.hq = r.hkv * a.G;
    r.q0 = 0;
    r.off = split;
    const int np = (a.P + BKV - 1) / BKV;
    r.p0 = split * t.split_blocks;
    r.np = min(t.split_blocks, np - r.p0);
    r.ns = r.wstart = r.light[0] = r.light[1] = 0;
    r.n_iter = r.np;
    r.live[0] = 1;
    r.live[1] = r.b + t.seqs_per_half < a.B;
    r.pre[0] = r.np;
    r.pre[1] = r.live[1] ? r.np : 0;
    r.wa[0] = r.wa[1] = 0;
    r.wb[0] = r.wb[1] = -1;
    return;
  }
  // heads in groups that fill the machine; inside a group the tiles from the last to the first, heads
  // innermost: a key head's blocks are in L2 while its query heads and neighbouring tiles read them
  const int BH = a.B * a.Hq;
  const int per_group = t.group_heads * t.n_qtiles;
  const int grp = idx / per_group, x = idx - grp * per_group;
  const int hg = min(BH - grp * t.group_heads, t.group_heads);
  const int bh = grp * t.group_heads + x % hg;
  r.q0 = (t.n_qtiles - 1 - x / hg) * BQ;
  r.b = bh / a.Hq;
  r.hq = bh % a.Hq;
  r.hkv = r.hq / a.G;
  r.off = len - a.Sq;
  int fw[2], lw[2];          // first and last own block that the rows' windows touch
  int wlo = 0x7fffffff, whi = -1, p_max = -1;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row0 = r.q0 + h * HALF;
    const int last = r.off + min(row0 + HALF, a.Sq) - 1;
    r.live[h] = row0 < a.Sq && last >= 0;
    fw[h] = max(max(r.off + row0, 0) - a.window + 1, 0) / BKV;
    lw[h] = last / BKV;
    if (r.live[h]) { wlo = min(wlo, fw[h]); whi = max(whi, lw[h]); p_max = max(p_max, last); }
    r.pre[h] = r.wa[h] = 0;
    r.wb[h] = -1;
  }
  r.p0 = r.np = r.ns = r.wstart = r.n_iter = r.light[0] = r.light[1] = 0;
  if (p_max >= 0) {
    r.np = (a.P + BKV - 1) / BKV;
    const bool few = r.np == 0 && a.sinks > 0 && a.sinks <= SINK_COLS;
    r.light[0] = few && r.live[0] && fw[0] > 0;
    r.light[1] = few && r.live[1] && fw[1] > 0;
    r.ns = (min(a.sinks, p_max + 1) + BKV - 1) / BKV;
    r.wstart = max(r.ns, wlo);
    r.n_iter = r.np + r.ns + max(whi - r.wstart + 1, 0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!r.live[h]) continue;
      r.pre[h] = r.np + min(r.ns, lw[h] + 1);
      r.wa[h] = r.np + r.ns + max(fw[h] - r.wstart, 0);
      r.wb[h] = r.np + r.ns + lw[h] - r.wstart;
    }
  }
}

// tile_ring entry: index (-1: no more) and the sequence's length
template <int HD, bool BF16, bool PACKED>
__global__ void __launch_bounds__(TA_THREADS, 1) tile_attention_kernel(const __grid_constant__ TileArgs t) {
  using L = TileSmem<HD>;
  const CacheAttn& a = t.a;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + B_COUNT);
  volatile int* tile_ring = reinterpret_cast<volatile int*>(bars + B_COUNT + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0 && lane == 0) {
    sm100::prefetch_tensormap(&t.tmap_q);
    if (!PACKED) sm100::prefetch_tensormap(&t.tmap_o);
    if (!PACKED && a.Skv > 0) { sm100::prefetch_tensormap(&t.tmap_k); sm100::prefetch_tensormap(&t.tmap_v); }
    if (a.P > 0) { sm100::prefetch_tensormap(&t.tmap_pk); sm100::prefetch_tensormap(&t.tmap_pv); }
    for (int i = 0; i < B_COUNT; ++i) {
      const bool per_warp = (i >= B_PFULL && i < B_PFULL + 2) || (i >= B_OFREE && i < B_OFREE + 2);
      const bool slot_free = i >= B_TEMPTY && i < B_TEMPTY + TILE_SLOTS;
      sm100::mbar_init(&bars[i], slot_free ? TILE_READERS : per_warp ? 4 : 1);
    }
    sm100::fence_barrier_init();
  }
  if (warp == 1) {
    sm100::tmem_alloc(tmem_slot, TMEM_COLS);
    sm100::tmem_relinquish();
  }
  if (PACKED) {
    // rows of a half above its box: no copy ever writes them, but the product reads them and their lanes have a say in
    // whether a warp takes a new reference maximum.  Zeros, so that the bits of the others depend on the inputs alone.
    const int box_rows = a.Sq * a.G * t.seqs_per_half, pieces = (128 - box_rows) * 8;   // 16 bytes each
    for (int x = threadIdx.x; x < 2 * (HD / 64) * pieces; x += TA_THREADS) {
      const int part = x / pieces, piece = x - part * pieces;                           // part: 64 columns of a half
      *reinterpret_cast<uint4*>(smem + L::Q_OFF + part * (128 * 128) + box_rows * 128 + piece * 16) = make_uint4(0, 0, 0, 0);
    }
    sm100::fence_proxy_async_smem();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // dependents start only after everything in front of this kernel is done (the streaming kernel behind the
  // packed prefix relies on it)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");

  if (warp < SOFTMAX_WARP0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONTROL));
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int ring = 0, loads = 0, q_loads = 0;
      bool ok = true;
      int idx = static_cast<int>(blockIdx.x);
      for (int k = 0; ok; ++k) {
        const int slot = k % TILE_SLOTS;
        const bool valid = idx < t.total_tiles;
        int len = 0;
        if (!PACKED && valid) {
          const int x = idx % (t.group_heads * t.n_qtiles), grp = idx / (t.group_heads * t.n_qtiles);
          const int hg = min(a.B * a.Hq - grp * t.group_heads, t.group_heads);
          len = sequence_length(a, (grp * t.group_heads + x % hg) / a.Hq);
        }
        if (k >= TILE_SLOTS && !sm100::mbar_wait(&bars[B_TEMPTY + slot], (k / TILE_SLOTS - 1) & 1)) { sm100::report_timeout(t.status, 40); break; }
        tile_ring[2 * slot] = valid ? idx : -1;
        tile_ring[2 * slot + 1] = len;
        sm100::mbar_arrive(&bars[B_TFULL + slot]);
        if (!valid) break;
        Tile r;
        decode_tile<PACKED>(t, idx, len, r);
        // packed tiles are alike and taken in turn; the others go to whoever is free
        idx = PACKED ? idx + static_cast<int>(gridDim.x) : t.next_tile ? static_cast<int>(gridDim.x + atomicAdd(t.next_tile, 1u)) : t.total_tiles;
        if (k > 0 && !sm100::mbar_wait(&bars[B_QEMPTY], (k - 1) & 1)) { sm100::report_timeout(t.status, 41); break; }
        const int q_bytes = PACKED ? a.Sq * a.G * t.seqs_per_half * HD * 2 : L::TILE_BYTES;
        sm100::mbar_arrive_expect_tx(&bars[B_QFULL], (r.live[0] + r.live[1]) * q_bytes);
        q_loads = k + 1;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (r.live[h])
#pragma unroll
            for (int d = 0; d < HD / 64; ++d)
              sm100::tma_load_4d(smem + L::Q_OFF + h * L::TILE_BYTES + d * (128 * 128), &t.tmap_q, d * 64,
                                 PACKED ? 0 : r.q0 + h * HALF, r.hq, PACKED ? r.b + h * t.seqs_per_half : r.b, &bars[B_QFULL]);
        for (int i = 0; i < 2 * r.n_iter; ++i) {      // K_j for i = 2j, V_j for i = 2j + 1
          const int n = ring + i, st = n % KV_STAGES, use = n / KV_STAGES, j = i >> 1;
          if (use > 0 && !sm100::mbar_wait(&bars[B_EMPTY + st], (use - 1) & 1)) { sm100::report_timeout(t.status, 42); ok = false; break; }
          sm100::mbar_arrive_expect_tx(&bars[B_FULL + st], L::TILE_BYTES);
          loads = n + 1;
          const bool pre = PACKED || j < r.np;
          const void* tmap = pre ? ((i & 1) ? static_cast<const void*>(&t.tmap_pv) : static_cast<const void*>(&t.tmap_pk))
                                 : ((i & 1) ? static_cast<const void*>(&t.tmap_v) : static_cast<const void*>(&t.tmap_k));
          const int key0 = (pre ? r.p0 + j : r.own_block(j)) * BKV;
#pragma unroll
          for (int d = 0; d < HD / 64; ++d)
            sm100::tma_load_4d(smem + L::KV_OFF + st * L::TILE_BYTES + d * (128 * 128), tmap, d * 64, key0, r.hkv, pre ? 0 : r.b,
                               &bars[B_FULL + st]);
        }
        ring += 2 * r.n_iter;
      }
      // no copy is in flight when the CTA ends, where a wait gave up either
      for (int n = max(loads - KV_STAGES, 0); n < loads; ++n) sm100::mbar_wait(&bars[B_FULL + n % KV_STAGES], (n / KV_STAGES) & 1);
      if (q_loads > 0) sm100::mbar_wait(&bars[B_QFULL], (q_loads - 1) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (convergent warp, elected lane)
    const bool leader = sm100::elect_one();
    constexpr uint32_t idesc_s = sm100::umma_idesc_f16(HALF, BKV, BF16, false, false);
    constexpr uint32_t idesc_light = sm100::umma_idesc_f16(HALF, SINK_COLS, BF16, false, false);
    constexpr uint32_t idesc_o = sm100::umma_idesc_f16(HALF, HD, BF16, false, true);  // V is MN-major
    auto wait_all = [&](uint64_t* bar, uint32_t parity, int site) -> bool {
      const bool done = __all_sync(0xffffffffu, sm100::mbar_wait(bar, parity));
      if (!done && leader) sm100::report_timeout(t.status, site);
      return done;
    };
    auto commit = [&](uint64_t* bar) {
      if (leader) sm100::umma_commit(bar);
      __syncwarp();
    };
    int ring = 0;
    int blocks[2] = {0, 0};       // key blocks issued so far per half (phases of its P barrier)
    int tiles_done[2] = {0, 0};   // tiles with at least one product issued, per half (gates the reuse of O_h)
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const int slot = k % TILE_SLOTS;
      ok = wait_all(&bars[B_TFULL + slot], (k / TILE_SLOTS) & 1, 43);
      if (!ok) break;
      // the reduction tells the compiler that all lanes hold the same tile: what follows from it (ring positions, operand
      // descriptors) then lives in uniform registers, where tcgen05.mma reads it
      const int idx = __reduce_max_sync(0xffffffffu, tile_ring[2 * slot]), len = __reduce_max_sync(0xffffffffu, tile_ring[2 * slot + 1]);
      __syncwarp();
      if (leader) sm100::mbar_arrive(&bars[B_TEMPTY + slot]);
      if (idx < 0) break;
      Tile r;
      decode_tile<PACKED>(t, idx, len, r);
      const int n_iter = r.n_iter;
      ok = wait_all(&bars[B_QFULL], k & 1, 44);
      if (!ok) break;
      auto ring_wait = [&](int i, int site) { const int n = ring + i; return wait_all(&bars[B_FULL + n % KV_STAGES], (n / KV_STAGES) & 1, site); };
      auto ring_free = [&](int i) { commit(&bars[B_EMPTY + (ring + i) % KV_STAGES]); };
      auto issue_s = [&](int h, int j, uint32_t idesc) {
        const uint32_t q_addr = sm100::smem_u32(smem + L::Q_OFF + h * L::TILE_BYTES);
        const uint32_t k_addr = sm100::smem_u32(smem + L::KV_OFF + ((ring + 2 * j) % KV_STAGES) * L::TILE_BYTES);
        const uint32_t d = tmem_base + TMEM_S + h * 128;
        const uint64_t qd = sm100::umma_desc_k_sw128(q_addr), kd = sm100::umma_desc_k_sw128(k_addr);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t o = ((kk / 4) * (128 * 128) + (kk % 4) * 32) >> 4;      // the address field counts 16 bytes
            sm100::umma_f16_ss(d, qd + o, kd + o, idesc, kk > 0 ? 1u : 0u);
          }
          sm100::umma_commit(&bars[B_SFULL + h]);
        }
        __syncwarp();
      };
      bool started[2] = {false, false};
      if (n_iter > 0) {
        ok = ring_wait(0, 45);
        if (!ok) break;
        sm100::tc_fence_after();
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (r.active(h, 0)) {
            if (!PACKED && r.light[h]) issue_s(h, 0, idesc_light);
            else issue_s(h, 0, idesc_s);
          }
        ring_free(0);
      }
      if (n_iter <= 1) commit(&bars[B_QEMPTY]);
      for (int j = 0; j < n_iter && ok; ++j) {
        const bool next = j + 1 < n_iter;
        const int vt = 2 * j + 1, kt = 2 * j + 2;
        ok = ring_wait(vt, 46);
        if (!ok) break;
        bool k_ready = false;
        unsigned char* v_tile = smem + L::KV_OFF + ((ring + vt) % KV_STAGES) * L::TILE_BYTES;
        const uint32_t v_addr = sm100::smem_u32(v_tile);
        if (!PACKED && !next && j >= r.np && len < a.Skv) {
          // the list ends with the block of the last position that some row of the tile sees.
          // V rows behind the sequence's end: a weight of 0 must not meet what the cache holds there
          const int keep = len - r.own_block(j) * BKV;
          if (keep < BKV) {
            for (int x = lane; x < (BKV - keep) * (HD / 8); x += 32) {
              const int row = keep + x / (HD / 8), piece = x % (HD / 8);
              *reinterpret_cast<uint4*>(v_tile + (piece >> 3) * (128 * 128) + row * 128 + (piece & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            sm100::fence_proxy_async_smem();
            __syncwarp();
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!ok) break;
          if (r.active(h, j)) {
            if (!started[h] && tiles_done[h] > 0) {    // the previous tile's epilogue must have read O_h
              ok = wait_all(&bars[B_OFREE + h], (tiles_done[h] - 1) & 1, 47);
              if (!ok) break;
            }
            ok = wait_all(&bars[B_PFULL + h], blocks[h] & 1, 48 + h);
            if (!ok) break;
            ++blocks[h];
            sm100::tc_fence_after();
            const uint32_t p_tmem = tmem_base + TMEM_S + h * 128;
            if (leader) {
              const uint32_t acc = started[h] ? 1u : 0u;
              const uint64_t vd = sm100::umma_desc_mn_sw128(v_addr, 128 * 128);
              auto products = [&](int steps) {
#pragma unroll
                for (int kk = 0; kk < steps; ++kk)
                  sm100::umma_f16_ts(tmem_base + TMEM_O + h * 128, p_tmem + kk * 8, vd + kk * ((16 * 128) >> 4), idesc_o, kk > 0 ? 1u : acc);
              };
              if (!PACKED && j == 0 && r.light[h]) products(SINK_COLS / 16);
              else products(BKV / 16);
              sm100::umma_commit(&bars[B_PVDONE + h]);
            }
            __syncwarp();
            if (!started[h]) { started[h] = true; ++tiles_done[h]; }
          }
          if (next && r.active(h, j + 1)) {
            if (!k_ready) {
              ok = ring_wait(kt, 50);
              if (!ok) break;
              k_ready = true;
              sm100::tc_fence_after();
            }
            issue_s(h, j + 1, idesc_s);
          }
        }
        if (!ok) break;
        ring_free(vt);
        if (next) {
          if (!k_ready && !(ok = ring_wait(kt, 50))) break;   // a stage is handed back only after it was filled
          ring_free(kt);
        }
        if (j + 2 == n_iter) commit(&bars[B_QEMPTY]);
      }
      ring += 2 * n_iter;
    }
    if (!ok) {                    // products in flight end before their tensor memory is freed
      commit(&bars[B_DRAIN]);
      sm100::mbar_wait(&bars[B_DRAIN], 0);
    }
  } else if (warp >= SOFTMAX_WARP0) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    // ------------------------------------------------------------ softmax / correction / epilogue
    const int g = (warp - SOFTMAX_WARP0) >> 2;       // half this warp group serves
    const int q = warp & 3;                          // tensor-memory lane quadrant
    const int row_in_half = q * 32 + lane;
    const uint32_t lane_sel = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t s_taddr = tmem_base + TMEM_S + g * 128 + lane_sel;
    const uint32_t o_taddr = tmem_base + TMEM_O + g * 128 + lane_sel;
    unsigned char* stage = smem + L::STAGE_OFF + (warp - SOFTMAX_WARP0) * L::WARP_STAGE;
    bool ok = true;      // a wait that gives up does so for the whole warp: what its lanes do together would wait for one that left
    int n = 0;                                       // key blocks consumed so far over all tiles
    for (int k = 0; ok; ++k) {
      const int slot = k % TILE_SLOTS;
      if (!__all_sync(0xffffffffu, sm100::mbar_wait(&bars[B_TFULL + slot], (k / TILE_SLOTS) & 1))) { sm100::report_timeout(t.status, 51); break; }
      const int idx = tile_ring[2 * slot], len = tile_ring[2 * slot + 1];
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&bars[B_TEMPTY + slot]);
      if (idx < 0) break;
      Tile r;
      decode_tile<PACKED>(t, idx, len, r);
      const int row0 = r.q0 + g * HALF;
      const int p_first = r.off + row0, p_last = r.off + min(row0 + HALF, a.Sq) - 1;
      const int pos = p_first + row_in_half;         // this row's position (PACKED: unused)
      const int warp_first = p_first + q * 32;       // and of the warp's first row
      // (selected, not indexed: an index that the compiler does not know would put the tile into local memory)
      const int live = g ? r.live[1] : r.live[0], light = g ? r.light[1] : r.light[0];
      const int pre = g ? r.pre[1] : r.pre[0], wa = g ? r.wa[1] : r.wa[0], wb = g ? r.wb[1] : r.wb[0];
      float m_ref = -INFINITY, l0 = 0.0f, l1 = 0.0f;
      bool first = true;

      for (int j = 0; j < r.n_iter; ++j) {
        if (j >= pre && (j < wa || j > wb)) continue;
        if (!__all_sync(0xffffffffu, sm100::mbar_wait(&bars[B_SFULL + g], n & 1))) { sm100::report_timeout(t.status, 52); ok = false; break; }
        ++n;
        sm100::tc_fence_after();
        if (!PACKED && j == 0 && light) {
          // sinks alone: 32 columns of scores, of which this row sees those in front of min(sinks, its position)
          first = false;
          softmax_sinks<BF16>(min(a.sinks, pos + 1), a.scale_log2, s_taddr, m_ref, l0);
          sm100::tmem_st_wait();
          sm100::tc_fence_before();
          __syncwarp();
          if (lane == 0) sm100::mbar_arrive(&bars[B_PFULL + g]);
          continue;
        }
        uint32_t sr[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) sm100::tmem_ld32(s_taddr + c * 32, sr[c]);
        sm100::tmem_ld_wait();

        if (PACKED || j < r.np) {
          const int left = a.P - (r.p0 + j) * BKV;   // keys of the prefix from here on
          if (left < BKV) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c * 32 + i >= left) sr[c][i] = __float_as_uint(-INFINITY);
          }
        } else {
          const int key0 = r.own_block(j) * BKV;
          if (key0 + BKV - 1 > p_first) {            // keys behind some row (behind the end too: p < len)
            const int see = pos - key0;              // visible: i <= see
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (key0 + c * 32 + 31 > warp_first)   // else every row of the warp sees the chunk
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (c * 32 + i > see) sr[c][i] = __float_as_uint(-INFINITY);
          }
          if (key0 <= p_last - a.window && key0 + BKV > a.sinks) {   // keys in front of some row's window
            const int gone = pos - a.window - key0;  // hidden: i <= gone, unless among the sinks
            if (key0 >= a.sinks) {
#pragma unroll
              for (int c = 0; c < 4; ++c)
                if (key0 + c * 32 <= warp_first + 31 - a.window)
#pragma unroll
                  for (int i = 0; i < 32; ++i)
                    if (c * 32 + i <= gone) sr[c][i] = __float_as_uint(-INFINITY);
            } else {
              const int sink = a.sinks - key0;
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (c * 32 + i <= gone && c * 32 + i >= sink) sr[c][i] = __float_as_uint(-INFINITY);
            }
          }
        }

        if (first) {
          first = false;
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              mx[i & 3] = max3(mx[i & 3], __uint_as_float(sr[c][2 * i]), __uint_as_float(sr[c][2 * i + 1]));
          m_ref = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), a.scale_log2, -WeightShift<BF16>::value);
          const float neg_m = (m_ref == -INFINITY) ? 0.0f : -m_ref;
          store_p<BF16, 0, false>(sr, a.scale_log2, neg_m, l0, l1, s_taddr);
        } else {
          float l0s = l0, l1s = l1;
          const float neg_m = (m_ref == -INFINITY) ? 0.0f : -m_ref;
          const float bmax = fmaf(store_p<BF16, 0, true>(sr, a.scale_log2, neg_m, l0s, l1s, s_taddr), a.scale_log2, -WeightShift<BF16>::value);
          if (__any_sync(0xffffffffu, bmax > m_ref + kRescale)) {
            const float m_new = fmaxf(m_ref, bmax);
            const float alpha = (m_ref == -INFINITY) ? 0.0f : fast_exp2(m_ref - m_new);
            l0 *= alpha;
            l1 *= alpha;
            m_ref = m_new;
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t o[32];
              sm100::tmem_ld32(o_taddr + c * 32, o);
              sm100::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              sm100::tmem_st32(o_taddr + c * 32, o);
            }
            sm100::tmem_st_wait();
            const float neg_m2 = (m_ref == -INFINITY) ? 0.0f : -m_ref;
            store_p<BF16, 0, false>(sr, a.scale_log2, neg_m2, l0, l1, s_taddr);
          } else {
            l0 = l0s;
            l1 = l1s;
          }
        }
        sm100::tmem_st_wait();
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&bars[B_PFULL + g]);
      }
      if (!ok) break;

      // ---- epilogue: O / l; O_h is handed back after the last read
      if (!live && (PACKED || row0 >= a.Sq)) continue;
      const float l = l0 + l1;
      const bool none = !live || (!PACKED && pos < 0) || l == 0.0f;
      const float inv = 1.0f / l;
      if (live) {
        if (!__all_sync(0xffffffffu, sm100::mbar_wait(&bars[B_PVDONE + g], (n - 1) & 1))) { sm100::report_timeout(t.status, 53); ok = false; break; }
        sm100::tc_fence_after();
      }
      if constexpr (PACKED) {
        // rows in packed order; 32 columns at a time through shared memory (16-byte pieces of a row XORed with the
        // row), so that four rows of 128 contiguous bytes leave with one instruction: a store per lane of its own
        // row touches 32 lines
        const int half_rows = a.G * a.Sq * t.seqs_per_half;
        const int64_t at = (static_cast<int64_t>(r.off) * a.Hkv + r.hkv) * t.part_rows + (r.b / t.seqs_per_half + g) * HALF;
        if (row_in_half < half_rows) t.part_lse[at + row_in_half] = none ? -INFINITY : m_ref + __log2f(l);
        unsigned char* part_stage = stage;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          sm100::tmem_ld32(o_taddr + c * 32, o);
          sm100::tmem_ld_wait();
          if (c == HD / 32 - 1) {
            sm100::tc_fence_before();
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&bars[B_OFREE + g]);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = none ? 0u : __float_as_uint(__uint_as_float(o[i]) * inv);
          __syncwarp();                              // the stage has been read
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(part_stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = i * 4 + (lane >> 3), piece = lane & 7;
            const uint4 v = *reinterpret_cast<const uint4*>(part_stage + row * 128 + ((piece ^ (row & 7)) << 4));
            if (q * 32 + row < half_rows) *reinterpret_cast<uint4*>(t.part_o + (at + q * 32 + row) * HD + c * 32 + piece * 4) = v;
          }
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t w[16];
          if (live) {
            uint32_t o[32];
            sm100::tmem_ld32(o_taddr + c * 32, o);
            sm100::tmem_ld_wait();
            if (c == HD / 32 - 1) {
              sm100::tc_fence_before();
              __syncwarp();
              if (lane == 0) sm100::mbar_arrive(&bars[B_OFREE + g]);
            }
#pragma unroll
            for (int x = 0; x < 16; ++x)
              w[x] = none ? 0u : pack_pair<BF16>(__uint_as_float(o[x * 2]) * inv, __uint_as_float(o[x * 2 + 1]) * inv);
          } else {
#pragma unroll
            for (int x = 0; x < 16; ++x) w[x] = 0u;    // a half of padding: nothing was computed
          }
          // two stages in turn, 64-byte swizzled (the lanes' 64-byte rows would meet in four banks)
          if (lane == 0) sm100::bulk_wait_read<1>();
          __syncwarp();
          unsigned char* out = stage + (c & 1) * (32 * 64);
#pragma unroll
          for (int x = 0; x < 4; ++x)
            *reinterpret_cast<uint4*>(out + lane * 64 + ((x ^ (lane >> 1 & 3)) << 4)) = make_uint4(w[x * 4], w[x * 4 + 1], w[x * 4 + 2], w[x * 4 + 3]);
          sm100::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            sm100::tma_store_4d(&t.tmap_o, out, c * 32, row0 + q * 32, r.hq, r.b);
            sm100::bulk_commit();
          }
        }
      }
    }
    if (!PACKED && lane == 0) sm100::bulk_wait<0>();
  }

  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------- host side
template <int HD, bool BF16, bool PACKED>
int launch_tile_cfg(TileArgs& t, int64_t tiles, int ctas, void* counter, cudaStream_t stream) {
  auto kern = tile_attention_kernel<HD, BF16, PACKED>;
  constexpr size_t smem = TileSmem<HD>::TOTAL;
  static bool configured_dev[64] = {false};
  int dev = 0;
  CDR_CUDA_TRY(cudaGetDevice(&dev));
  if (!configured_dev[dev & 63]) {
    // setmaxnreg.inc waits until the CTA's registers at launch cover the split: refuse a build that got fewer
    cudaFuncAttributes fa;
    CDR_CUDA_TRY(cudaFuncGetAttributes(&fa, kern));
    if (fa.numRegs * TA_THREADS < 128 * REGS_CONTROL + (TA_THREADS - 128) * REGS_SOFTMAX) {
      set_error("attention: kernel was built with %d registers per thread, fewer than its register split needs", fa.numRegs);
      return CDR_ERR_UNSUPPORTED;
    }
    CDR_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    configured_dev[dev & 63] = true;
  }
  t.total_tiles = static_cast<int>(tiles);
  t.status = device_status_ptr();
  const int64_t grid = tiles < ctas ? tiles : ctas;
  t.next_tile = nullptr;
  if (!PACKED && tiles > grid) { // CTAs draw tiles beyond their first from a counter
    t.next_tile = static_cast<unsigned int*>(counter);
    CDR_CUDA_TRY(cudaMemsetAsync(t.next_tile, 0, sizeof(unsigned int), stream));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(TA_THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CDR_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, t));
  return CDR_OK;
}

template <bool PACKED>
int launch_tile_typed(TileArgs& t, int64_t tiles, int ctas, void* counter, cudaStream_t stream) {
  if (tiles > 0x3fffffff) { set_error("attention: too many tiles"); return CDR_ERR_UNSUPPORTED; }
  if (t.a.D == 128) return t.a.bf16 ? launch_tile_cfg<128, true, PACKED>(t, tiles, ctas, counter, stream) : launch_tile_cfg<128, false, PACKED>(t, tiles, ctas, counter, stream);
  return t.a.bf16 ? launch_tile_cfg<64, true, PACKED>(t, tiles, ctas, counter, stream) : launch_tile_cfg<64, false, PACKED>(t, tiles, ctas, counter, stream);
}

int map_heads(CUtensorMap* m, const void* base, const CacheAttn& a, int64_t S, int64_t H, int64_t B, const HeadStrides& st, int box_d,
              int box_s, int box_h, int box_b, int swizzle_bytes) {
  const int64_t dims[4] = {a.D, S, H, B}, strides[3] = {st.s, st.h, st.b};
  const int box[4] = {box_d, box_s, box_h, box_b};
  return make_tensor_map_4d(m, base, a.bf16, dims, strides, box, swizzle_bytes);
}

int map_prefix(TileArgs& t) {
  const CacheAttn& a = t.a;
  if (a.P == 0) return CDR_OK;
  HeadStrides pk = a.spk, pv = a.spv;
  pk.b = pv.b = a.D;             // one "sequence": the stride is never used
  if (int rc = map_heads(&t.tmap_pk, a.pk, a, a.P, a.Hkv, 1, pk, 64, BKV, 1, 1, 128)) return rc;
  return map_heads(&t.tmap_pv, a.pv, a, a.P, a.Hkv, 1, pv, 64, BKV, 1, 1, 128);
}

}  // namespace

float tile_attention_us(const CacheAttn& a) {
  const int64_t keys = static_cast<int64_t>(a.window) + (a.Sq < BQ ? a.Sq : BQ);
  const int64_t own = (a.Skv + BKV - 1) / BKV, touched = ((keys < a.Skv ? keys : a.Skv) + 2 * BKV - 1) / BKV;
  const int64_t sinks = ((a.sinks < a.Skv ? a.sinks : a.Skv) + BKV - 1) / BKV;      // in front of the window, as far as there are keys
  const int64_t blocks = (touched + sinks < own + 1 ? touched + sinks : own + 1) + (a.P + BKV - 1) / BKV;
  const int64_t tiles = static_cast<int64_t>(a.B) * a.Hq * ((a.Sq + BQ - 1) / BQ);
  return 6.0f + (a.D == 128 ? 2.0f : 1.7f) * ((tiles + sm_count() - 1) / sm_count()) * blocks;
}

int launch_tile_attention(const CacheAttn& a, void* ws, cudaStream_t stream) {
  TileArgs t = {};
  t.a = a;
  if (int rc = map_heads(&t.tmap_q, a.q, a, a.Sq, a.Hq, a.B, a.sq, 64, HALF, 1, 1, 128)) return rc;
  if (int rc = map_heads(&t.tmap_o, a.out, a, a.Sq, a.Hq, a.B, a.so, 32, 32, 1, 1, 64)) return rc;
  if (a.Skv > 0) {               // an empty cache is never loaded from
    if (int rc = map_heads(&t.tmap_k, a.k, a, a.Skv, a.Hkv, a.B, a.sk, 64, BKV, 1, 1, 128)) return rc;
    if (int rc = map_heads(&t.tmap_v, a.v, a, a.Skv, a.Hkv, a.B, a.sv, 64, BKV, 1, 1, 128)) return rc;
  }
  if (int rc = map_prefix(t)) return rc;
  t.n_qtiles = (a.Sq + BQ - 1) / BQ;
  const int64_t BH = static_cast<int64_t>(a.B) * a.Hq;
  if (BH * t.n_qtiles > 0x3fffffff) { set_error("attention: too many tiles"); return CDR_ERR_UNSUPPORTED; }
  const int fill = sm_count() / t.n_qtiles;
  t.group_heads = static_cast<int>(fill < 1 ? 1 : fill > BH ? BH : fill);
  return launch_tile_typed<false>(t, BH * t.n_qtiles, sm_count(), ws, stream);
}

// How the shared prefix is cut for the packed product, and how many CTAs it gets: the others of the machine's
// SMs are left to the streaming kernel, which starts beside it (own keys from HBM under the product's arithmetic).
// Both times are estimated, in us, from what the kernels measure on this machine: here 1.95 per block of 128 keys and 256
// rows (1.6 with one live half, a fifth less at D = 64), 3 per tile and 5 per launch; there 0.19 per 16 KB and SM, 8 per launch.  64 sequences of 32
// heads behind 16384 keys, 512 own ones: 71 us one after the other, 46.6 with 88 CTAs here, 52.9 with 112, 72 with 120.
PackedPlan plan_packed(const CacheAttn& a, int64_t own_units) {
  PackedPlan p;
  const int per_seq = a.G * a.Sq;
  const int fit = HALF / per_seq;
  p.seqs_per_half = fit < a.B ? fit : a.B;
  p.row_tiles = (a.B + 2 * p.seqs_per_half - 1) / (2 * p.seqs_per_half);
  const int blocks = (a.P + BKV - 1) / BKV;
  const int64_t tasks = static_cast<int64_t>(a.Hkv) * p.row_tiles;
  const int sms = sm_count();
  const float per_block = (p.seqs_per_half < a.B ? 1.95f : 1.6f) * (a.D == 128 ? 1.0f : 0.8f);
  const float stream_us = 0.19f * own_units * a.D / 128;
  float best = INFINITY;
  for (int eighth = 4; eighth <= 8; ++eighth) {
    const int ctas = ((eighth == 8 ? sms - sms / 16 : sms * eighth / 8) + 3) / 4 * 4;
    for (int rounds = 1; rounds <= 2; ++rounds) {
      int64_t splits = rounds * ctas / tasks;
      splits = splits < 1 ? 1 : splits > blocks ? blocks : splits;
      const int split_blocks = static_cast<int>((blocks + splits - 1) / splits);
      splits = (blocks + split_blocks - 1) / split_blocks;
      const float tile_us = 5.0f + (tasks * splits + ctas - 1) / ctas * (split_blocks * per_block + 3.0f);
      const float us = fmaxf(tile_us, 8.0f + stream_us / (sms > ctas ? sms - ctas : 1));
      if (us < best) {
        best = us;
        p.split_blocks = split_blocks;
        p.splits = static_cast<int>(splits);
        p.ctas = static_cast<int>(tasks * splits < ctas ? tasks * splits : ctas);
      }
    }
  }
  p.us = best + 6.0f;            // and the parts are added up
  return p;
}

size_t packed_workspace(const CacheAttn& a, const PackedPlan& p) {
  return static_cast<size_t>(p.splits) * a.Hkv * p.row_tiles * 2 * HALF * (a.D + 1) * sizeof(float);
}

int launch_packed_prefix(const CacheAttn& a, const PackedPlan& plan, void* ws, PrefixPartials* part, cudaStream_t stream) {
  TileArgs t = {};
  t.a = a;
  t.seqs_per_half = plan.seqs_per_half;
  t.n_qtiles = plan.row_tiles;
  t.split_blocks = plan.split_blocks;
  t.splits = plan.splits;
  const int64_t rows = static_cast<int64_t>(plan.row_tiles) * 2 * HALF;
  if (rows > 0x3fffffff) { set_error("attention: too many sequences"); return CDR_ERR_UNSUPPORTED; }
  t.part_rows = static_cast<int>(rows);
  t.part_o = static_cast<float*>(ws);
  t.part_lse = t.part_o + static_cast<size_t>(t.splits) * a.Hkv * rows * a.D;
  if (int rc = map_heads(&t.tmap_q, a.q, a, a.Sq, a.Hq, a.B, a.sq, 64, a.Sq, a.G, t.seqs_per_half, 128)) return rc;
  if (int rc = map_prefix(t)) return rc;
  *part = PrefixPartials{t.part_o, t.part_lse, t.splits, t.part_rows, t.seqs_per_half};
  return launch_tile_typed<true>(t, static_cast<int64_t>(t.splits) * a.Hkv * t.n_qtiles, plan.ctas, nullptr, stream);
}

}  // namespace cdr
