// Attention of many rows a request over the paged 8-bit cache (quant8.cuh) on the 5th-generation tensor cores, for heads of 64
// and 128 (-DLAB_HEAD_DIM): portions of prompts.
//
// Two kernels.  The first turns the keys and values that a portion's rows see into bfloat16, once (exactly: a code has four
// significant bits, a scale is a power of two), in the order of the keys, into scratch: every tile of rows walks the same keys,
// and turning them anew in each CTA cost more than the attention's own arithmetic (measured, below).  The second is the
// attention over those rows:
//
// A CTA takes 128 rows of one request and kv head and walks the keys in tiles of 128.  Row r is token r / group and query head
// r % group of those that share the kv head, so a tile of keys is fetched once for all of them, and a CTA's rows reach over few
// positions: only the last tiles of its walk (and a window's first) need a mask.
//   S = Q K^T       kind::f16, from shared memory
//   P = softmax(S)  a thread a row: mask, running maximum and sum in 32 bits, 2^x, P rounded to bfloat16 into tensor memory
//   O += P V        P from tensor memory
// Two groups of four warps take the tiles in turn, even and odd ones, each a thread a row of the same 128 rows.  Tensor memory
// holds two S, two P and the one O: the scores of a group's next tile are formed as soon as it has read the present ones, so
// that no group waits for the tensor cores, and neither do they for a group.  (Two groups with rows, S, P over S and O of their
// own instead: a tile of 128 keys and 256 rows took 4,450 cycles, of which 1,700 went into the signals between the warps
// alone, and none of the ways to shorten them helped: 64 keys a tile, two threads a row, fewer registers.)
// The groups share a row's reference maximum, to which O is relative: a group decides on it for its tile after the other has
// for the tile before, which it learns through shared memory.  The reference follows the maximum only when that has grown by
// more than 2^32 (two portions of 1,024 rows: a tenth less time than with 2^8, where some row of a warp's 32 grows in most of the
// first tiles; no bit is lost by it, P and O being floating-point numbers; only values beyond 2^95 or so can take O out of its
// range), and O is then rescaled in place, the product of the tile before being complete.  Each group keeps a sum of its own.
//
// A key that is no number is a row of NaN, and so is one whose value is none (its value then 0): the rows that see it become
// NaN, and no others.  Rows behind the last key are 0.
//
// Where the rows make fewer CTAs than the GPU holds (a portion of a few hundred rows behind a long context), the keys are split over
// CTAs: each leaves its O, reference and sum in scratch, and a third kernel joins them.
//
// The exponentials and the warps' signals bound it, beside tensor cores that are active 45 % of the time (two portions of 1,024 rows,
// 28 + 4 heads of 128, a window of 4,096: 137 us with the first kernel's 14, 755 TFLOP/s).
//
// Warps: 0 loads (TMA), 1 issues the scores' products, 2 those with V, 4-7 and 8-11 are the groups.  setmaxnreg: 384 threads of
// 168 registers become 232 a softmax thread and 40 the rest: 2 x 232 + 40 = 3 x 168.  Every wait is bounded.
#include "quant8_tc.cuh"

#ifndef LAB_HEAD_DIM
#error "build with -DLAB_HEAD_DIM=64 or 128"
#endif

namespace {

constexpr int D = LAB_HEAD_DIM;
constexpr int KEYS = 128, ROWS = 128, GROUPS = 2, THREADS = 384;
constexpr int STAGES = D == 64 ? 4 : 3;
constexpr int HALVES = D / 64, HALF_BYTES = KEYS * 128;      // swizzled tiles of 64 columns, 128 bytes a row
constexpr int TILE = HALVES * HALF_BYTES;                    // 128 rows
constexpr int OFF_Q = 0;
constexpr int OFF_K = OFF_Q + TILE;
constexpr int OFF_V = OFF_K + STAGES * TILE;
constexpr int OFF_ROW = OFF_V + STAGES * TILE;               // a row's reference maximum, and its two sums
constexpr int OFF_BAR = OFF_ROW + 3 * ROWS * 4;
constexpr int SMEM = OFF_BAR + 384 + 1024;
static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
constexpr int TM_S = 0, TM_P = GROUPS * KEYS, TM_O = TM_P + GROUPS * KEYS / 2, TMEM_COLS = 512;
static_assert(TM_O + D <= TMEM_COLS, "tensor memory holds two S, two P and one O");
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE = 32.f;      // P and O have an exponent of eight bits: up to 2^32 too large they are as exact (values below 2^95)

struct Barriers {
  uint64_t q_full, k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[GROUPS], s_empty[GROUPS], p_full[GROUPS],
      o_full[GROUPS], turn[GROUPS][4];
  uint32_t tmem_slot;
  int abort_flag;
};
static_assert(sizeof(Barriers) <= 384, "barriers fit their place");

struct Args {
  __nv_bfloat16* out;
  long long out_stride;
  const __nv_bfloat16* q;
  long long q_stride;
  const uint8_t *k, *v, *k_scale, *v_scale;
  const int *q_start, *kv_len, *pos0, *block_table;
  int tokens, max_blocks, request0, requests, look0, look1, n_q, n_kv, page_size, num_pages, window, fewest, longest, many;
  __nv_bfloat16 *wide_k, *wide_v;      // [requests of many rows][n_kv][span][D]
  int span;                            // keys, a multiple of KEYS
  int splits;                          // of the keys of a tile of rows
  float* part;                         // of a split: [D + 2][ROWS], the entries of O, the reference and the sum of each row
  float scale_log2;
};

// A request's keys in scratch start at the tile of the first that its rows see.
__device__ __forceinline__ int first_tile(int pos0, int window) { return lab_first_key(pos0, window) / KEYS; }
// The grids have a slice (z) for each of the `many` requests of many rows that the host has counted, not for every request: beside one
// portion 63 single tokens made 63 slices of CTAs that found nothing to do (a portion of 2,048 rows, 14 + 2 heads of 64: 120 us with the
// few-rows kernel's 11, 42 now; 28 + 4 heads of 128: 264 with 37, 117 now).  Slice z belongs to the z-th of them, -1 where the device's
// counts have no such; by one warp, all its lanes get it.  Where all requests of a run have many rows (MIXED false) no lookup is
// needed: builds of their own, since a lookup's loads and code cost about 1 us (2,048 rows beside one token: 40.1 us, 38.9 without; two
// portions of 1,024 rows of 28 + 4 heads 137.8, 137.3).
template <bool MIXED> __device__ __forceinline__ int request_of(const Args& a, int z, int lane) {
  if constexpr (MIXED) {
    int left = z;
    for (int i0 = 0; i0 < a.requests; i0 += 32) {
      const int i = a.request0 + i0 + lane;
      const uint32_t found = __ballot_sync(0xffffffffu, i0 + lane < a.requests && a.q_start[i + 1] - a.q_start[i] >= a.fewest);
      const int here = __popc(found);
      if (left < here) return a.request0 + i0 + (int)__fns(found, 0, left + 1);
      left -= here;
    }
    return -1;
  } else {
    return a.request0 + z;
  }
}

// The place of a request's keys and values in scratch: its number among those of many rows.  (Also where that is the slice's as a rule: so
// the attention's loop keeps the registers it had, 8,192 rows of 14 + 2 heads of 64 in 193 us, 200 with z itself.)
template <bool MIXED> __device__ __forceinline__ int place_of(const Args& a, int b, int z, int lane) {
  if constexpr (MIXED) return z;
  int n = 0;
  for (int i = a.request0 + lane; i < b; i += 32) n += a.q_start[i + 1] - a.q_start[i] >= a.fewest;
  return __reduce_add_sync(0xffffffffu, n);
}

// Whether a request is within what the host has been told: its rows among the batch's, its keys within a request's scratch.
__device__ __forceinline__ bool within(const Args& a, int qs, int ql, int p0, int last) {
  return qs >= 0 && qs <= a.tokens - ql && ql <= a.longest && last < first_tile(p0, a.window) * KEYS + a.span;
}

// Where a split of a tile of rows leaves its results: `tiles` tiles a request and kv head.
__device__ __forceinline__ float* part_of(const Args& a, int place, int tile, int tiles, int kvh, int split) {
  return a.part + ((((size_t)place * tiles + tile) * a.n_kv + kvh) * a.splits + split) * ((D + 2) * ROWS);
}

// ----------------------------------------------------------------------------------------
// Codes to bfloat16: a CTA a tile of keys of one request and kv head, 16 codes of a key and 16 of a value a thread and turn.
// ----------------------------------------------------------------------------------------
constexpr int WIDEN_THREADS = 256;
template <bool MIXED>
__global__ void __launch_bounds__(WIDEN_THREADS) widen_kernel(const Args a) {
  pdl_trigger();
  pdl_wait();
  const int kvh = blockIdx.y, lane = threadIdx.x & 31;
  // Requests of many rows for which there is no slice, from look0 up to look1: one warp of the launch looks for such.
  if (blockIdx.x == 0 && kvh == 0 && blockIdx.z == 0 && threadIdx.x >= WIDEN_THREADS - 32) {
    int left = a.many;      // of the slices
    for (int i = a.look0 + lane; i - lane < a.look1; i += 32) {
      const bool many = i < a.look1 && a.q_start[i + 1] - a.q_start[i] >= a.fewest, inside = i >= a.request0 && i < a.request0 + a.requests;
      left -= __popc(__ballot_sync(0xffffffffu, many && inside));
      if (__any_sync(0xffffffffu, many && !inside)) left = -1;
      if (left < 0) break;
    }
    if (left < 0 && lane == 0) lab_set_error(LAB_ERR_ROW_RANGE);
  }
  const int b = request_of<MIXED>(a, blockIdx.z, lane);
  if (MIXED && b < 0) return;
  const int qs = a.q_start[b], ql = a.q_start[b + 1] - qs;
  if (ql < a.fewest) return;
  const int p0 = a.pos0[b], first = lab_first_key(p0, a.window);
  const int last = min(min(p0 + ql, a.kv_len[b]), a.max_blocks * a.page_size) - 1;
  const int key0 = (first_tile(p0, a.window) + (int)blockIdx.x) * KEYS;
  if (!within(a, qs, ql, p0, last)) {
    if (threadIdx.x == 0) lab_set_error(LAB_ERR_ROW_RANGE);
    return;
  }
  if (key0 > last) return;
  const int* bt = a.block_table + (size_t)b * a.max_blocks;
  const size_t to0 = (((size_t)place_of<MIXED>(a, b, blockIdx.z, lane) * a.n_kv + kvh) * a.span + (size_t)blockIdx.x * KEYS) * D;
  constexpr int PIECES = D / 16, TURNS = KEYS * PIECES / WIDEN_THREADS;
  static_assert(KEYS * PIECES % WIDEN_THREADS == 0, "whole turns");
  uint4 kc[TURNS], vc[TURNS];
  float ks[TURNS], vs[TURNS];
#pragma unroll
  for (int t = 0; t < TURNS; ++t) {      // all loads of a thread in flight together
    const int e = t * WIDEN_THREADS + threadIdx.x, j = key0 + e / PIECES, piece = e % PIECES;
    kc[t] = vc[t] = make_uint4(0, 0, 0, 0);
    ks[t] = vs[t] = 0.f;
    if (j < first || j > last) continue;
    const int page = bt[j / a.page_size];
    if (page < 0 || page >= a.num_pages) {      // a page that holds visible keys must exist
      lab_set_error(LAB_ERR_PAGE_RANGE);
      continue;
    }
    const size_t at = ((size_t)page * a.n_kv + kvh) * a.page_size + j % a.page_size;
    kc[t] = *reinterpret_cast<const uint4*>(a.k + at * D + piece * 16);
    vc[t] = *reinterpret_cast<const uint4*>(a.v + at * D + piece * 16);
    const uint32_t kb = a.k_scale[at], vb = a.v_scale[at];
    ks[t] = q8_scale(vb == Q8_NAN_BYTE ? Q8_NAN_BYTE : kb);
    vs[t] = vb == Q8_NAN_BYTE ? 0.f : q8_scale(vb);
  }
#pragma unroll
  for (int t = 0; t < TURNS; ++t) {
    const int e = t * WIDEN_THREADS + threadIdx.x;
    auto put = [&](__nv_bfloat16* out, const uint4& c, float f) {
      const uint32_t w[4] = {c.x, c.y, c.z, c.w};
      uint32_t r[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 x = q8_decode4(w[i]);
        r[2 * i] = pack_bf16(x.x * f, x.y * f), r[2 * i + 1] = pack_bf16(x.z * f, x.w * f);
      }
      uint4* to = reinterpret_cast<uint4*>(out + to0 + (size_t)(e / PIECES) * D + (e % PIECES) * 16);
      to[0] = make_uint4(r[0], r[1], r[2], r[3]);
      to[1] = make_uint4(r[4], r[5], r[6], r[7]);
    };
    put(a.wide_k, kc[t], ks[t]);
    put(a.wide_v, vc[t], vs[t]);
  }
}

__device__ __forceinline__ float max_of(float a, float b, float c) {      // (a NaN is passed over)
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <bool MIXED>
__global__ void __launch_bounds__(THREADS, 1) attention_q8_rows_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                       const __grid_constant__ CUtensorMap map_v, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  Barriers* bar = reinterpret_cast<Barriers*>(smem + OFF_BAR);
  volatile int* abort_flag = &bar->abort_flag;
  pdl_trigger();
  // Until pdl_wait() below only the step's metadata is read (no kernel of the step writes it).
  // kv heads fastest, a request's last rows first: the CTAs that walk the most keys start in the first wave
  const int split = blockIdx.x / a.n_kv, kvh = blockIdx.x - split * a.n_kv, group = a.n_q / a.n_kv;
  const int b = request_of<MIXED>(a, blockIdx.z, threadIdx.x & 31);
  if (MIXED && b < 0) {
    pdl_wait();  // this kernel ends only after the one before it: what follows may count on both
    return;
  }
  const int qs = a.q_start[b], ql = a.q_start[b + 1] - qs;
  const int r0 = (gridDim.y - 1 - blockIdx.y) * ROWS;
  const int p0 = a.pos0[b];
  if (ql < a.fewest || r0 >= ql * group || !within(a, qs, ql, p0, min(min(p0 + ql, a.kv_len[b]), a.max_blocks * a.page_size) - 1)) {
    pdl_wait();
    return;
  }
  // The warp's number from one lane, so that the compiler sees a warp's branches as its lanes' common ones: for heads of 128 alone (two
  // portions of 1,024 rows: 134.7 us, 140.4 without; heads of 64: 74.9 and 70.7, 8,192 rows 178 and 165).
  const int warp = D == 128 ? __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0) : (int)(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int last_row = min(r0 + ROWS, ql * group) - 1;
  const int pos_lo = p0 + r0 / group, pos_hi = p0 + last_row / group;
  const int last = min(min(pos_hi, a.kv_len[b] - 1), a.max_blocks * a.page_size - 1), first = lab_first_key(pos_lo, a.window);
  const int all_tiles = last >= first ? last / KEYS - first / KEYS + 1 : 0, each = all_tiles / a.splits, more = all_tiles - each * a.splits;
  const int t_lo = first / KEYS + split * each + min(split, more), n_tiles = each + (split < more ? 1 : 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&bar->k_full[s], 1);
      mbar_init(&bar->k_empty[s], 1);
      mbar_init(&bar->v_full[s], 1);
      mbar_init(&bar->v_empty[s], 1);
    }
    mbar_init(&bar->q_full, 4);
    for (int g = 0; g < GROUPS; ++g) {
      mbar_init(&bar->s_full[g], 1);
      mbar_init(&bar->s_empty[g], 4);
      mbar_init(&bar->p_full[g], 4);
      mbar_init(&bar->o_full[g], 1);
      for (int w = 0; w < 4; ++w) mbar_init(&bar->turn[g][w], 1);
    }
    bar->abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc(&bar->tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem_base = bar->tmem_slot, smem_base = smem_u32(smem);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      // ---------------- loader ----------------
      const int row0 = (place_of<MIXED>(a, b, blockIdx.z, lane) * a.n_kv + kvh) * a.span + (t_lo - first_tile(p0, a.window)) * KEYS;
      if (lane == 0) {
        int asked = 0;
        for (int j = 0; j < n_tiles; ++j) {
          const int s = j % STAGES;
          const uint32_t ph = (j / STAGES) & 1;
          if (!mbar_wait(&bar->k_empty[s], ph ^ 1, abort_flag)) break;
          mbar_expect_tx(&bar->k_full[s], TILE);
          for (int hf = 0; hf < HALVES; ++hf)
            tma_load_2d(smem_base + OFF_K + s * TILE + hf * HALF_BYTES, &map_k, &bar->k_full[s], hf * 64, row0 + j * KEYS);
          asked = 2 * j + 1;
          if (!mbar_wait(&bar->v_empty[s], ph ^ 1, abort_flag)) break;
          mbar_expect_tx(&bar->v_full[s], TILE);
          for (int hf = 0; hf < HALVES; ++hf)
            tma_load_2d(smem_base + OFF_V + s * TILE + hf * HALF_BYTES, &map_v, &bar->v_full[s], hf * 64, row0 + j * KEYS);
          asked = 2 * j + 2;
        }
        if (asked < 2 * n_tiles) {      // a wait has run out: the copies that were asked for land before the CTA ends
          volatile int never = 0;
          for (int i = max(0, asked - 2 * STAGES); i < asked; ++i) {
            const int j = i / 2, s = j % STAGES;
            mbar_wait(i & 1 ? &bar->v_full[s] : &bar->k_full[s], (j / STAGES) & 1, &never, 100000000ull);
          }
        }
      }
    } else if (warp == 1) {
      // ---------------- scores: a group's next as soon as it has read the present ones ----------------
      constexpr uint32_t idesc = umma_instr_desc(ROWS, KEYS);
      bool ok = n_tiles > 0 && mbar_wait(&bar->q_full, 0, abort_flag);
      for (int j = 0; j < n_tiles; ++j) {
        const int s = j % STAGES, g = j & 1;
        ok = ok && mbar_wait(&bar->k_full[s], (j / STAGES) & 1, abort_flag) && mbar_wait(&bar->s_empty[g], ((j >> 1) & 1) ^ 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
#pragma unroll
        for (int hf = 0; hf < HALVES; ++hf) {
          const uint64_t qd = smem_desc_sw128(smem_base + OFF_Q + hf * HALF_BYTES), kd = smem_desc_sw128(smem_base + OFF_K + s * TILE + hf * HALF_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16(tmem_base + TM_S + g * KEYS, qd + 2 * k, kd + 2 * k, idesc, (hf | k) > 0);
        }
        umma_commit(&bar->s_full[g]);
        umma_commit(&bar->k_empty[s]);
      }
    } else if (warp == 2) {
      // ---------------- P V: as soon as P is there (a warp of its own: neither kind of product waits for the other's operands) ----------------
      constexpr uint32_t idesc = umma_instr_desc(ROWS, D, true);
      bool ok = true;
      for (int j = 0; j < n_tiles; ++j) {
        const int s = j % STAGES, g = j & 1;
        ok = mbar_wait(&bar->v_full[s], (j / STAGES) & 1, abort_flag) && mbar_wait(&bar->p_full[g], (j >> 1) & 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const uint64_t vd = q8_desc(smem_base + OFF_V + s * TILE, HALF_BYTES, 1024, 2);
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k)      // 16 keys of V lie 16 rows of 128 bytes on
          umma_bf16_tmem_a(tmem_base + TM_O, tmem_base + TM_P + g * (KEYS / 2) + k * 8, vd + (uint64_t)(k * 16 * 128 / 16), idesc, (k | j) > 0);
        umma_commit(&bar->o_full[g]);
        umma_commit(&bar->v_empty[s]);
      }
    }
  } else {
    // ---------------- softmax: a thread a row, a group every other tile ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int g = (warp - 4) >> 2, quarter = warp & 3, mine = quarter * 32 + lane;
    const int r = r0 + mine, token = r / group, head = kvh * group + r - token * group;
    const bool valid = r < ql * group;
    const int pos = p0 + token, hi = valid ? min(pos, last) : -1, lo = lab_first_key(pos, a.window);
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    if (g == 0) {
      const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)(qs + token) * a.q_stride + (size_t)head * D);
      uint8_t* q_s = smem + OFF_Q + mine * 128;
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        *reinterpret_cast<uint4*>(q_s + (c >> 3) * HALF_BYTES + ((c & 7) ^ (mine & 7)) * 16) = valid ? src[c] : make_uint4(0, 0, 0, 0);
      proxy_fence();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->q_full);
    }
    const uint32_t s_addr = lane_addr + TM_S + g * KEYS, p_addr = lane_addr + TM_P + g * (KEYS / 2), o_addr = lane_addr + TM_O;
    const f32x2 factor2 = pair_of(a.scale_log2, a.scale_log2);
    volatile float* reference = reinterpret_cast<volatile float*>(smem + OFF_ROW) + mine;      // then the two sums, ROWS further each
    float m_ref = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = g; j < n_tiles; j += GROUPS) {
      const uint32_t phase = (j >> 1) & 1;
      ok = mbar_wait(&bar->s_full[g], phase, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[KEYS];
#pragma unroll
      for (int c = 0; c < KEYS / 32; ++c) tmem_ld32_issue(s_addr + c * 32, sr + c * 32);
      tmem_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->s_empty[g]);
      // Two conditions that hold by now as a rule are asked for here and looked at when they are needed: the other group has
      // decided for the tile before, and this group's P of two tiles ago has been multiplied (and with it all before that).
      const bool decided = j == 0 || mbar_try_wait(&bar->turn[g][quarter], ((j - 1) >> 1) & 1);
      const bool multiplied = j < GROUPS || mbar_try_wait(&bar->o_full[g], phase ^ 1);
      const int key0 = (t_lo + j) * KEYS;
      if (!__all_sync(0xffffffffu, key0 >= lo && key0 + KEYS - 1 <= hi)) {
        const int from = lo - key0, to = hi - key0;
#pragma unroll
        for (int c = 0; c < KEYS; ++c)
          if (c < from || c > to) sr[c] = __float_as_uint(-INFINITY);
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < KEYS; c += 2) mx4[(c >> 1) & 3] = max_of(mx4[(c >> 1) & 3], __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
      const float top = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2;
      float m_old = -INFINITY;
      if (!__all_sync(0xffffffffu, decided && multiplied)) {
        if (!decided) ok = mbar_wait(&bar->turn[g][quarter], ((j - 1) >> 1) & 1, abort_flag);
        if (!multiplied) ok = mbar_wait(&bar->o_full[g], phase ^ 1, abort_flag) && ok;
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      if (j > 0) m_old = *reference;
      const float m_top = fmaxf(m_old, top);
      const bool grows = __any_sync(0xffffffffu, m_top > m_old + RESCALE || (m_old == -INFINITY && m_top != -INFINITY));
      const float m_new = grows ? m_top : m_old;
      *reference = m_new;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->turn[g ^ 1][quarter]);
      l *= m_ref == m_new ? 1.f : fast_exp2(m_ref - m_new);
      m_ref = m_new;
      if (grows && j > 0) {
        ok = mbar_wait(&bar->o_full[g ^ 1], ((j - 1) >> 1) & 1, abort_flag);      // and that of the tile before
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const float f = m_old == m_new ? 1.f : fast_exp2(m_old - m_new);
#pragma unroll
        for (int part = 0; part < D / 16; ++part) {
          uint32_t o[16];
          tmem_ld16_issue(o_addr + part * 16, o);
          tmem_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
          tmem_st16(o_addr + part * 16, o);
        }
      }
      const float base = m_ref == -INFINITY ? 0.f : m_ref;
      const f32x2 base2 = pair_of(-base, -base);
      f32x2 sum2[2] = {0ull, 0ull};
#pragma unroll
      for (int c = 0; c < KEYS / 32; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const f32x2 e = fma2(pair_of(__uint_as_float(sr[c * 32 + 2 * i]), __uint_as_float(sr[c * 32 + 2 * i + 1])), factor2, base2);
          const float p = fast_exp2(low_of(e)), q = fast_exp2(high_of(e));
          sum2[i & 1] = add2(sum2[i & 1], pair_of(p, q));
          pk[i] = pack_bf16(p, q);
        }
        tmem_st16(p_addr + c * 16, pk);
      }
      const f32x2 sum = add2(sum2[0], sum2[1]);
      l += low_of(sum) + high_of(sum);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->p_full[g]);
    }
    // The row's sum: each group's, relative to the last reference.
    if (ok && n_tiles > 0) {
      if (((n_tiles - 1) & 1) != g) ok = mbar_wait(&bar->turn[g][quarter], ((n_tiles - 1) >> 1) & 1, abort_flag);
      const float m_last = *reference;
      l *= m_ref == m_last ? 1.f : fast_exp2(m_ref - m_last);
    }
    reference[(1 + g) * ROWS] = l;
    asm volatile("bar.sync 1, 256;" ::: "memory");      // (a group that has given up comes here too)
    l += reference[(1 + (g ^ 1)) * ROWS];
    if (n_tiles > 0) {      // (all lanes of a warp come to the vote: one that has given up may have done so alone)
      ok = ok && mbar_wait(&bar->o_full[(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok && a.splits > 1) {      // half of the head's entries a group, neighbouring rows side by side
      tc_fence_after();
      float* to = part_of(a, blockIdx.z, gridDim.y - 1 - blockIdx.y, gridDim.y, kvh, split) + mine;
#pragma unroll
      for (int part = 0; part < D / 64; ++part) {
        uint32_t x[32];
        tmem_ld32_issue(o_addr + g * (D / 2) + part * 32, x);
        tmem_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          to[(g * (D / 2) + part * 32 + i) * ROWS] = n_tiles == 0 ? 0.f : __uint_as_float(x[i]);
      }
      if (g == 0) to[D * ROWS] = n_tiles == 0 ? -INFINITY : *reference, to[(D + 1) * ROWS] = l;
    } else if (ok) {      // half of the head's entries a group
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      __nv_bfloat16* dst = a.out + (size_t)(qs + token) * a.out_stride + (size_t)head * D + g * (D / 2);
#pragma unroll
      for (int part = 0; part < D / 64; ++part) {
        uint32_t x[32];
        __syncwarp();
        tmem_ld32_issue(o_addr + g * (D / 2) + part * 32, x);   // every lane takes part in the load
        tmem_wait();
        if (!valid) continue;
        auto number = [&](int i) { return n_tiles == 0 ? 0.f : __uint_as_float(x[i]) * inv; };
#pragma unroll
        for (int q8 = 0; q8 < 4; ++q8) {
          const uint4 packed = make_uint4(pack_bf16(number(8 * q8), number(8 * q8 + 1)), pack_bf16(number(8 * q8 + 2), number(8 * q8 + 3)),
                                          pack_bf16(number(8 * q8 + 4), number(8 * q8 + 5)), pack_bf16(number(8 * q8 + 6), number(8 * q8 + 7)));
          __nv_bfloat16* d8 = dst + part * 32 + q8 * 8;
          if ((((uintptr_t)d8) & 15) == 0) {
            *reinterpret_cast<uint4*>(d8) = packed;
          } else {
            const __nv_bfloat16* hp = reinterpret_cast<const __nv_bfloat16*>(&packed);
            for (int e = 0; e < 8; ++e) d8[e] = hp[e];
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// The splits of a tile of rows put together: a thread a row and MERGED entries of the head, neighbouring threads neighbouring rows, 16
// bytes a store (two portions of 256 rows over 3,000 keys in three: 33 us with the call's other kernels, 59 with 2 bytes a store).
constexpr int MERGED = 8;
template <bool MIXED>
__global__ void __launch_bounds__(ROWS, 6) attention_q8_rows_merge_kernel(const Args a) {
  pdl_trigger();
  pdl_wait();
  const int piece = blockIdx.x / a.n_kv, kvh = blockIdx.x - piece * a.n_kv, group = a.n_q / a.n_kv;
  const int b = request_of<MIXED>(a, blockIdx.z, threadIdx.x & 31);
  if (MIXED && b < 0) return;
  const int qs = a.q_start[b], ql = a.q_start[b + 1] - qs, p0 = a.pos0[b], r = blockIdx.y * ROWS + threadIdx.x;
  if (ql < a.fewest || r >= ql * group || !within(a, qs, ql, p0, min(min(p0 + ql, a.kv_len[b]), a.max_blocks * a.page_size) - 1)) return;
  float m = -INFINITY, den = 0.f, num[MERGED];
#pragma unroll
  for (int i = 0; i < MERGED; ++i) num[i] = 0.f;
  const float* from = part_of(a, blockIdx.z, blockIdx.y, gridDim.y, kvh, 0) + threadIdx.x;
  constexpr int STEP = (D + 2) * ROWS;      // to the next split
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, from[s * STEP + D * ROWS]);
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float ms = from[s * STEP + D * ROWS], f = ms == -INFINITY ? 0.f : fast_exp2(ms - m);
    den = fmaf(f, from[s * STEP + (D + 1) * ROWS], den);      // (0 times a NaN is one: scores that are all none stay visible)
#pragma unroll
    for (int i = 0; i < MERGED; ++i) num[i] = fmaf(f, from[s * STEP + (piece * MERGED + i) * ROWS], num[i]);
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const int token = r / group, head = kvh * group + r - token * group;
  __nv_bfloat16* dst = a.out + (size_t)(qs + token) * a.out_stride + (size_t)head * D + piece * MERGED;
  uint32_t packed[MERGED / 2];
#pragma unroll
  for (int i = 0; i < MERGED / 2; ++i) packed[i] = pack_bf16(num[2 * i] * inv, num[2 * i + 1] * inv);
  if ((((uintptr_t)dst) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < MERGED / 8; ++i)
      reinterpret_cast<uint4*>(dst)[i] = make_uint4(packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
  } else {
    const __nv_bfloat16* each = reinterpret_cast<const __nv_bfloat16*>(packed);
#pragma unroll
    for (int i = 0; i < MERGED; ++i) dst[i] = each[i];
  }
}

// Keys that a request's rows reach over at most, whole tiles and one more for where the first begins.
int span_of(int window, int most_keys, int longest) {
  const int w = window < 0 ? -window : window;
  const long long keys = window == 0 ? most_keys : (long long)w + longest < most_keys ? (long long)w + longest : most_keys;
  return (int)((keys + KEYS - 1) / KEYS + 1) * KEYS;
}

template <bool MIXED>
int launch_rows(const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, int tiles, cudaStream_t stream) {
  static LabShared granted;
  cudaError_t e = lab_allow_shared(granted, (const void*)attention_q8_rows_kernel<MIXED>, SMEM);
  if (e != cudaSuccess) return (int)e;
  e = lab_launch(widen_kernel<MIXED>, dim3(a.span / KEYS, a.n_kv, a.many), dim3(WIDEN_THREADS), 0, stream, a);
  if (e != cudaSuccess) return (int)e;
  e = lab_launch(attention_q8_rows_kernel<MIXED>, dim3(a.n_kv * a.splits, tiles, a.many), dim3(THREADS), (size_t)SMEM, stream, mk, mv, a);
  if (e != cudaSuccess || a.splits == 1) return (int)e;
  return (int)lab_launch(attention_q8_rows_merge_kernel<MIXED>, dim3(a.n_kv * (D / MERGED), tiles, a.many), dim3(ROWS), 0, stream, a);
}

}  // namespace

// Bytes of scratch for `many` requests of many rows, whose longest brings `longest` and whose lengths are at most most_keys.
LAB_EXPORT long long lab_attention_q8_rows_scratch(int many, int n_kv, int window, int most_keys, int longest) {
  return (long long)many * n_kv * span_of(window, most_keys, longest) * D * 4;
}

// Bytes of scratch for the splits' results of a call, none with one.
LAB_EXPORT long long lab_attention_q8_rows_parts(int many, int n_kv, int group, int longest, int splits) {
  return splits < 2 ? 0 : (long long)many * (((long long)longest * group + ROWS - 1) / ROWS) * n_kv * splits * (D + 2) * ROWS * 4;
}

// A call, as the host packs it.  q: `tokens` rows q_stride elements apart, on 16-byte boundaries, out likewise; the `requests` from
// request0 on, those of `fewest` rows or more (shorter ones are left alone), `many` of them, `longest` the most rows that one
// brings; others of that many rows among the requests from look0 up to look1 are reported; lengths are at most most_keys; scratch on a
// boundary of 16 bytes.  splits: CTAs that share the keys of a tile of rows, their results in `parts` where there are several.  window as
// lab_first_key takes it.
struct LabQ8Rows {
  void* out;
  const void *q, *k, *v, *k_scale, *v_scale;
  const int *q_start, *kv_len, *pos0, *block_table;
  void *scratch, *parts;
  long long out_stride, q_stride;
  int tokens, max_blocks, request0, requests, look0, look1, n_q, n_kv, page_size, num_pages, window, fewest, longest, many, most_keys, splits;
  float scale;
};

LAB_EXPORT int lab_attention_q8_rows(const LabQ8Rows* c, cudaStream_t stream) {
  if (c->requests <= 0 || c->longest <= 0 || c->many <= 0) return 0;
  const int span = span_of(c->window, c->most_keys, c->longest);
  const long long rows = (long long)c->many * c->n_kv * span;
  if (c->n_kv < 1 || c->n_q < 1 || c->n_q % c->n_kv || c->max_blocks < 1 || c->num_pages < 1 || c->fewest < 1 || c->page_size < 1 || c->request0 < 0 ||
      c->splits < 1 || (c->splits > 1 && (c->parts == nullptr || (((uintptr_t)c->parts) & 3))) || (long long)c->n_kv * c->splits >= (1ll << 31) ||
      c->most_keys < 1 || rows >= (1ll << 31) || c->many > c->requests || c->look0 < 0 || c->many > 65535 || c->n_kv > 65535 || c->q_stride % 8 || (((uintptr_t)c->q) & 15) ||
      ((((uintptr_t)c->k) | ((uintptr_t)c->v) | ((uintptr_t)c->scratch)) & 15) || c->scratch == nullptr)
    return (int)cudaErrorInvalidValue;
  Args a;
  a.out = (__nv_bfloat16*)c->out, a.out_stride = c->out_stride, a.q = (const __nv_bfloat16*)c->q, a.q_stride = c->q_stride;
  a.k = (const uint8_t*)c->k, a.v = (const uint8_t*)c->v, a.k_scale = (const uint8_t*)c->k_scale, a.v_scale = (const uint8_t*)c->v_scale;
  a.q_start = c->q_start, a.kv_len = c->kv_len, a.pos0 = c->pos0, a.block_table = c->block_table, a.max_blocks = c->max_blocks;
  a.n_q = c->n_q, a.n_kv = c->n_kv, a.page_size = c->page_size, a.num_pages = c->num_pages, a.window = c->window, a.fewest = c->fewest;
  a.tokens = c->tokens, a.request0 = c->request0, a.requests = c->requests, a.look0 = c->look0, a.look1 = c->look1, a.longest = c->longest, a.many = c->many;
  a.wide_k = (__nv_bfloat16*)c->scratch, a.wide_v = a.wide_k + (size_t)rows * D, a.span = span;
  a.splits = c->splits, a.part = (float*)c->parts, a.scale_log2 = c->scale * LOG2E;
  CUtensorMap mk, mv;
  int rc;
  if ((rc = lab_make_map_bf16(&mk, a.wide_k, rows, D, D, KEYS))) return rc;
  if ((rc = lab_make_map_bf16(&mv, a.wide_v, rows, D, D, KEYS))) return rc;
  const long long tiles = ((long long)c->longest * (c->n_q / c->n_kv) + ROWS - 1) / ROWS;
  if (tiles > 65535) return (int)cudaErrorInvalidValue;
  return c->many < c->requests ? launch_rows<true>(mk, mv, a, (int)tiles, stream) : launch_rows<false>(mk, mv, a, (int)tiles, stream);
}
