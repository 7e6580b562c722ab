// Attention of many rows a request over the paged 8-bit cache (quant8.cuh) on the 5th-generation tensor cores, for heads of 64
// and 128 (-DLAB_HEAD_DIM) and pages of 8 to 128 tokens: portions of prompts.
//
// A CTA takes 256 rows of one request and kv head, two groups of 128, and walks the keys in tiles of 128.  Row r is token r /
// group and query head r % group of those that share the kv head, so a tile of keys is fetched and converted once for all of
// them, and a CTA's rows reach over few positions: only the last tiles of its walk need a mask.
//   S = Q K^T       kind::f8f6f4, K as cached.  A row of q, after a power of two, is cut into two codes whose sum it is
//                   (quant8_tc.cuh): two products of 8-bit operands take the time of one of 16-bit ones, and nothing of K is converted
//   P = softmax(S)  a thread a row: scores times their keys' scales (powers of two, broadcast from shared memory), mask, running
//                   maximum and sum in 32 bits, 2^x, P rounded to bfloat16 over the scores in tensor memory
//   O += P V        kind::f16, P from tensor memory, V from shared memory as bfloat16
// V is converted, not cut: four warps turn a tile's codes and scales into bfloat16 (exactly: a code has four significant bits)
// while the tensor cores are busy with the others.  Two codes of P instead would have to be formed by the softmax threads, which
// are what bounds the kernel, and reach down to 2^-18 of the row's maximum only.  O accumulates in tensor memory relative to a
// reference maximum and is rescaled only when a row's maximum has grown by more than 2^8.  A group's scores follow its own P V in
// the tensor cores' queue, so scores that have arrived say that O is complete: the two groups take turns, one at its softmax
// while the products of the other run.
//
// Warps: 0 loads (TMA, a page a lane), 1 issues the products, 4-7 convert (a thread a key), 8-11 and 12-15 are the groups.
// setmaxnreg: 512 threads of 128 registers become 192 a softmax thread, 72 a converting one, 56 the rest: 2 x 192 + 72 + 56 =
// 4 x 128.  Every wait is bounded.
#include "quant8_tc.cuh"

#ifndef LAB_HEAD_DIM
#error "build with -DLAB_HEAD_DIM=64 or 128"
#endif

namespace {

constexpr int D = LAB_HEAD_DIM;
using Tile = Q8Tile<D>;
constexpr int KEYS = Tile::KEYS, ROWS = 128, GROUPS = 2, THREADS = 512;
constexpr int STAGES = D == 64 ? 4 : 2;
constexpr int HALVES = D / 64, HALF_BYTES = KEYS * 128;      // V as bfloat16: swizzled tiles of 64 columns, 128 bytes a key
constexpr int VB_BYTES = HALVES * HALF_BYTES;
constexpr int OFF_Q = 0;                                     // [group][high, low][128, D]
constexpr int OFF_K = OFF_Q + GROUPS * 2 * ROWS * D;
constexpr int OFF_V = OFF_K + STAGES * Tile::BYTES;
constexpr int OFF_VB = OFF_V + STAGES * Tile::BYTES;
constexpr int OFF_KS = OFF_VB + 2 * VB_BYTES;                // [2][128] floats: the keys' scales
constexpr int OFF_BAR = OFF_KS + 2 * KEYS * 4;
constexpr int SMEM = OFF_BAR + 256 + 1024;
static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
constexpr int TM_S = 0, TM_O = GROUPS * KEYS, TMEM_COLS = 512;
static_assert(TM_O + GROUPS * D <= TMEM_COLS, "tensor memory holds two S and two O");
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE = 8.f;

struct Barriers {
  uint64_t q_full[GROUPS], k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], ks_full[2], vb_full[2], vb_empty[2],
      s_full[GROUPS], p_full[GROUPS], o_full[GROUPS];
  uint32_t tmem_slot;
  int abort_flag;
};
static_assert(sizeof(Barriers) <= 256, "barriers fit their place");

struct Args {
  __nv_bfloat16* out;
  long long out_stride;
  const __nv_bfloat16* q;
  long long q_stride;
  const uint8_t *k_scale, *v_scale;
  const int *q_start, *kv_len, *pos0, *block_table;
  int max_blocks, n_q, n_kv, page_size, num_pages, window, fewest;
  float scale_log2;
};

// Four codes to bfloat16, in the order 0, 2, 1, 3: the codes' bits at a bfloat16's places are the numbers times 2^-120
// (subnormal ones included), and `times` is 2^120 and more.
__device__ __forceinline__ uint2 widen4(uint32_t w, __nv_bfloat162 times) {
  const uint32_t up = w << 8;
  uint32_t even = ((up & 0x7f007f00u) >> 4) | (up & 0x80008000u), odd = ((w & 0x7f007f00u) >> 4) | (w & 0x80008000u);
  __nv_bfloat162 a = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&even), times), b = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&odd), times);
  return make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}
__device__ __forceinline__ __nv_bfloat162 power_pair(int exponent) {      // 2^exponent twice
  const uint32_t bits = (uint32_t)(exponent + 127) << 7, both = bits | bits << 16;
  return *reinterpret_cast<const __nv_bfloat162*>(&both);
}

__global__ void __launch_bounds__(THREADS, 1) attention_q8_rows_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                       const __grid_constant__ CUtensorMap map_v, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  Barriers* bar = reinterpret_cast<Barriers*>(smem + OFF_BAR);
  volatile int* abort_flag = &bar->abort_flag;
  pdl_trigger();
  // kv heads fastest, a request's last rows first: the CTAs that walk the most keys start in the first wave
  const int b = blockIdx.z, kvh = blockIdx.x, group = a.n_q / a.n_kv;
  const int qs = a.q_start[b], ql = a.q_start[b + 1] - qs;
  const int r0 = (gridDim.y - 1 - blockIdx.y) * (GROUPS * ROWS);
  if (ql < a.fewest || r0 >= ql * group) {
    pdl_wait();  // this kernel ends only after the one before it: what follows may count on both
    return;
  }
  const int p0 = a.pos0[b], kvl = a.kv_len[b];
  const int* bt = a.block_table + (size_t)b * a.max_blocks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int last_row = min(r0 + GROUPS * ROWS, ql * group) - 1;
  const int pos_lo = p0 + r0 / group, pos_hi = p0 + last_row / group;
  const int last = min(min(pos_hi, kvl - 1), a.max_blocks * a.page_size - 1), first = lab_first_key(pos_lo, a.window);
  const int t_lo = first / KEYS, n_tiles = last >= first ? last / KEYS - t_lo + 1 : 0;
  const int page_shift = __ffs(a.page_size) - 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&bar->k_full[s], 1);
      mbar_init(&bar->k_empty[s], 1);
      mbar_init(&bar->v_full[s], 1);
      mbar_init(&bar->v_empty[s], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->ks_full[i], 4);
      mbar_init(&bar->vb_full[i], 4);
      mbar_init(&bar->vb_empty[i], 1);
      mbar_init(&bar->q_full[i], 4);
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->p_full[i], 4);
      mbar_init(&bar->o_full[i], 1);
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // ---------------- loader: a page a lane ----------------
      const int pages_per_tile = KEYS >> page_shift, page_bytes = D << page_shift;
      auto page_row = [&](int j) -> int {      // the pool's row of this lane's page in tile j, -1: not fetched
        if (j >= n_tiles || lane >= pages_per_tile) return -1;
        const int k_lo = (t_lo + j) * KEYS + (lane << page_shift);
        if (k_lo > last || k_lo + a.page_size <= first) return -1;
        const int page = bt[k_lo >> page_shift];
        if (page >= a.num_pages || page < 0) {      // a page that holds visible keys must exist
          lab_set_error(LAB_ERR_PAGE_RANGE);
          return -1;
        }
        return (page * a.n_kv + kvh) << page_shift;
      };
      int next = page_row(0), asked = 0;
      for (int j = 0; j < n_tiles; ++j) {
        const int s = j % STAGES;
        const uint32_t ph = (j / STAGES) & 1;
        const int row = next;
        next = page_row(j + 1);
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, row >= 0)) * page_bytes;
        const bool alive = mbar_wait(&bar->k_empty[s], ph ^ 1, abort_flag) && mbar_wait(&bar->v_empty[s], ph ^ 1, abort_flag);
        if (!__all_sync(0xffffffffu, alive)) break;
        if (lane == 0) {
          mbar_expect_tx(&bar->k_full[s], bytes);
          mbar_expect_tx(&bar->v_full[s], bytes);
        }
        __syncwarp();
        if (row >= 0) {
          tma_load_2d(smem_base + OFF_K + s * Tile::BYTES + lane * page_bytes, &map_k, &bar->k_full[s], 0, row);
          tma_load_2d(smem_base + OFF_V + s * Tile::BYTES + lane * page_bytes, &map_v, &bar->v_full[s], 0, row);
        }
        asked = j + 1;
      }
      if (asked < n_tiles) {      // a wait has run out: the copies that were asked for land before the CTA ends
        volatile int never = 0;
        for (int j = max(0, asked - STAGES); j < asked; ++j) {
          mbar_wait(&bar->k_full[j % STAGES], (j / STAGES) & 1, &never, 100000000ull);
          mbar_wait(&bar->v_full[j % STAGES], (j / STAGES) & 1, &never, 100000000ull);
        }
      }
    } else if (warp == 1) {
      // ---------------- products ----------------
      constexpr uint32_t idesc_s = q8_instr(ROWS, KEYS, false, false), idesc_o = umma_instr_desc(ROWS, D, true);
      auto wait_all = [&](uint64_t* m, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(m, parity, abort_flag)); };
      auto issue_s = [&](int j, int g) {
        const uint64_t kd = q8_desc(smem_base + OFF_K + (j % STAGES) * Tile::BYTES, 16, Tile::GROUP, Tile::LAYOUT);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint64_t qd = q8_desc(smem_base + OFF_Q + (g * 2 + half) * ROWS * D, 16, Tile::GROUP, Tile::LAYOUT);
#pragma unroll
          for (int k = 0; k < D / 32; ++k) umma_q8(tmem_base + TM_S + g * KEYS, qd + 2 * k, kd + 2 * k, idesc_s, (half | k) > 0);
        }
        umma_commit(&bar->s_full[g]);
      };
      bool ok = n_tiles > 0 && wait_all(&bar->k_full[0], 0);
      for (int g = 0; g < GROUPS && ok; ++g) {
        ok = wait_all(&bar->q_full[g], 0);
        tc_fence_after();
        if (ok) issue_s(0, g);
      }
      if (ok) umma_commit(&bar->k_empty[0]);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int t = j & 1;
        ok = wait_all(&bar->vb_full[t], (j >> 1) & 1);
        const uint64_t vd = q8_desc(smem_base + OFF_VB + t * VB_BYTES, HALF_BYTES, 1024, 2);
        for (int g = 0; g < GROUPS && ok; ++g) {
          ok = wait_all(&bar->p_full[g], j & 1);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < KEYS / 16; ++k)      // 16 keys of V lie 16 rows of 128 bytes on
            umma_bf16_tmem_a(tmem_base + TM_O + g * D, tmem_base + TM_S + g * KEYS + k * 8, vd + (uint64_t)(k * 16 * 128 / 16), idesc_o,
                             (k | j) > 0);
          if (j + 1 < n_tiles) {
            if (g == 0) ok = wait_all(&bar->k_full[(j + 1) % STAGES], ((j + 1) / STAGES) & 1);
            if (!ok) break;
            tc_fence_after();
            issue_s(j + 1, g);
          } else {
            umma_commit(&bar->o_full[g]);
          }
        }
        if (!ok) break;
        umma_commit(&bar->vb_empty[t]);
        if (j + 1 < n_tiles) umma_commit(&bar->k_empty[(j + 1) % STAGES]);
      }
    }
  } else if (warp < 8) {
    // ---------------- values to bfloat16, and the keys' scales: a thread a key ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int mine = (warp - 4) * 32 + lane;
    float* ks_s = reinterpret_cast<float*>(smem + OFF_KS);
    auto row_of = [&](int j) -> long long {
      if (j < first || j > last) return -1;
      const int page = bt[j >> page_shift];
      return page < 0 || page >= a.num_pages ? -1 : (((long long)page * a.n_kv + kvh) << page_shift) + (j & (a.page_size - 1));
    };
    long long row = n_tiles > 0 ? row_of(t_lo * KEYS + mine) : -1;
    uint32_t kb = row >= 0 ? a.k_scale[row] : 127, vb = row >= 0 ? a.v_scale[row] : 127;
    for (int j = 0; j < n_tiles; ++j) {
      const int s = j % STAGES, t = j & 1;
      const bool held = row >= 0;
      // a value that is no number counts as a score that is none; its place in V, as that of a key that is not there, is 0
      const float ks = !held ? 0.f : vb == Q8_NAN_BYTE ? q8_scale(Q8_NAN_BYTE) : q8_scale(kb);
      const int power = (int)vb - 127;
      const bool zero = !held || vb == Q8_NAN_BYTE;
      if (j + 1 < n_tiles) {      // the next key's bytes arrive beside this tile
        row = row_of((t_lo + j + 1) * KEYS + mine);
        kb = row >= 0 ? a.k_scale[row] : 127, vb = row >= 0 ? a.v_scale[row] : 127;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&bar->vb_empty[t], ((j >> 1) & 1) ^ 1, abort_flag))) break;
      ks_s[t * KEYS + mine] = ks;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->ks_full[t]);
      if (!__all_sync(0xffffffffu, mbar_wait(&bar->v_full[s], (j / STAGES) & 1, abort_flag))) break;
      // 2^(120 + power) in one factor up to power 7 (values beyond 57,344), in two above
      const __nv_bfloat162 times = zero ? __floats2bfloat162_rn(0.f, 0.f) : power_pair(max(-126, min(127, 120 + power)));
      const bool large = __any_sync(0xffffffffu, !zero && power > 7);
      const __nv_bfloat162 more = power_pair(max(0, power - 7));
      const uint8_t* from = smem + OFF_V + s * Tile::BYTES;
      uint8_t* to = smem + OFF_VB + t * VB_BYTES + mine * 128;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(from + Tile::piece_at(mine, c));
        uint2 x[4] = {widen4(w.x, times), widen4(w.y, times), widen4(w.z, times), widen4(w.w, times)};
        if (large) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&x[i]);
            p[0] = __hmul2(p[0], more), p[1] = __hmul2(p[1], more);
          }
        }
        uint8_t* half = to + (c >> 2) * HALF_BYTES;
        *reinterpret_cast<uint4*>(half + (((2 * c) & 7) ^ (mine & 7)) * 16) = make_uint4(x[0].x, x[0].y, x[1].x, x[1].y);
        *reinterpret_cast<uint4*>(half + (((2 * c + 1) & 7) ^ (mine & 7)) * 16) = make_uint4(x[2].x, x[2].y, x[3].x, x[3].y);
      }
      proxy_fence();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bar->v_empty[s]);
        mbar_arrive(&bar->vb_full[t]);
      }
    }
  } else {
    // ---------------- softmax: a thread a row ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int g = (warp - 8) >> 2, quarter = warp & 3, mine = quarter * 32 + lane;
    const int r = r0 + g * ROWS + mine, token = r / group, head = kvh * group + r - token * group;
    const bool valid = r < ql * group;
    const int pos = p0 + token, hi = valid ? min(pos, last) : -1, lo = lab_first_key(pos, a.window);
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    float factor = 0.f;
    {
      // q: a power of two, and two codes
      uint4 x[D / 8];
#pragma unroll
      for (int c = 0; c < D / 8; ++c) x[c] = make_uint4(0, 0, 0, 0);
      if (valid) {
        const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)(qs + token) * a.q_stride + (size_t)head * D);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) x[c] = src[c];
      }
      uint32_t top = 0;      // of the numbers' upper 16 bits
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fff0000u, (w[i] << 16) & 0x7fff0000u));
      }
      const int byte = q8_byte(top);
      const float inverse = byte == Q8_NAN_BYTE ? 0.f : q8_inverse(byte);
      factor = valid ? a.scale_log2 * q8_scale(byte) : 0.f;
      uint8_t* q_s = smem + OFF_Q + g * 2 * ROWS * D;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        uint32_t high[4], low[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 v = x[2 * c + (i >> 1)];
          const uint32_t w0 = (i & 1) ? v.z : v.x, w1 = (i & 1) ? v.w : v.y;
          float f[4] = {__uint_as_float(w0 << 16) * inverse, __uint_as_float(w0 & 0xffff0000u) * inverse, __uint_as_float(w1 << 16) * inverse,
                        __uint_as_float(w1 & 0xffff0000u) * inverse};
          if (byte == Q8_NAN_BYTE) f[0] = f[1] = f[2] = f[3] = 0.f;
          q8_split4(f, high[i], low[i]);
        }
        *reinterpret_cast<uint4*>(q_s + Tile::piece_at(mine, c)) = make_uint4(high[0], high[1], high[2], high[3]);
        *reinterpret_cast<uint4*>(q_s + ROWS * D + Tile::piece_at(mine, c)) = make_uint4(low[0], low[1], low[2], low[3]);
      }
      proxy_fence();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->q_full[g]);
    }
    const uint32_t s_addr = lane_addr + TM_S + g * KEYS, o_addr = lane_addr + TM_O + g * D;
    const float* ks_s = reinterpret_cast<const float*>(smem + OFF_KS);
    float m_ref = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      ok = mbar_wait(&bar->ks_full[j & 1], (j >> 1) & 1, abort_flag) && mbar_wait(&bar->s_full[g], j & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[KEYS];
#pragma unroll
      for (int c = 0; c < KEYS / 32; ++c) tmem_ld32_issue(s_addr + c * 32, sr + c * 32);
      tmem_wait();
      const float4* ks4 = reinterpret_cast<const float4*>(ks_s + (j & 1) * KEYS);
      const int key0 = (t_lo + j) * KEYS;
#pragma unroll
      for (int c = 0; c < KEYS / 4; ++c) {
        const float4 f = ks4[c];
        const f32x2 x = mul2(pair_of(__uint_as_float(sr[4 * c]), __uint_as_float(sr[4 * c + 1])), pair_of(f.x, f.y));
        const f32x2 y = mul2(pair_of(__uint_as_float(sr[4 * c + 2]), __uint_as_float(sr[4 * c + 3])), pair_of(f.z, f.w));
        sr[4 * c] = __float_as_uint(low_of(x)), sr[4 * c + 1] = __float_as_uint(high_of(x));
        sr[4 * c + 2] = __float_as_uint(low_of(y)), sr[4 * c + 3] = __float_as_uint(high_of(y));
      }
      if (!__all_sync(0xffffffffu, key0 >= lo && key0 + KEYS - 1 <= hi)) {
#pragma unroll
        for (int c = 0; c < KEYS; ++c)
          if (key0 + c < lo || key0 + c > hi) sr[c] = __float_as_uint(-INFINITY);
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < KEYS; ++c) mx4[c & 3] = fmaxf(mx4[c & 3], __uint_as_float(sr[c]));
      const float top = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      const float m_new = top == -INFINITY ? m_ref : fmaxf(m_ref, top * factor);      // (a factor may be 0, or no number)
      if (j == 0) {
        m_ref = m_new;
      } else if (__any_sync(0xffffffffu, m_new > m_ref + RESCALE || (m_ref == -INFINITY && m_new != -INFINITY))) {
        const float f = m_ref == m_new ? 1.f : fast_exp2(m_ref - m_new);
#pragma unroll
        for (int part = 0; part < D / 32; ++part) {
          uint32_t x[32];
          tmem_ld32_issue(o_addr + part * 32, x);
          tmem_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
          tmem_st32(o_addr + part * 32, x);
        }
        l *= f;
        m_ref = m_new;
      }
      const float base = m_ref == -INFINITY ? 0.f : m_ref;
      const f32x2 factor2 = pair_of(factor, factor), base2 = pair_of(-base, -base);
      float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c32 = 0; c32 < KEYS / 64; ++c32) {
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int c = c32 * 64 + 2 * i;
          const f32x2 e = fma2(pair_of(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), factor2, base2);
          const float x = fast_exp2(low_of(e)), y = fast_exp2(high_of(e));
          sum4[i & 1] += x;
          sum4[2 + (i & 1)] += y;
          pk[i] = pack_bf16(x, y);
        }
        tmem_st32(s_addr + c32 * 32, pk);
      }
      l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->p_full[g]);
    }
    if (ok && n_tiles > 0) {
      ok = mbar_wait(&bar->o_full[g], 0, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      __nv_bfloat16* dst = a.out + (size_t)(qs + token) * a.out_stride + (size_t)head * D;
#pragma unroll
      for (int part = 0; part < D / 32; ++part) {
        uint32_t x[32];
        tmem_ld32_issue(o_addr + part * 32, x);   // every lane takes part in the load
        tmem_wait();
        if (!valid) continue;
        auto number = [&](int i) { return n_tiles == 0 ? 0.f : __uint_as_float(x[i]) * inv; };
#pragma unroll
        for (int q8 = 0; q8 < 4; ++q8) {      // (columns lie in the order of `widen4`)
          const uint4 packed = make_uint4(pack_bf16(number(8 * q8), number(8 * q8 + 2)), pack_bf16(number(8 * q8 + 1), number(8 * q8 + 3)),
                                          pack_bf16(number(8 * q8 + 4), number(8 * q8 + 6)), pack_bf16(number(8 * q8 + 5), number(8 * q8 + 7)));
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

}  // namespace

// Requests of `fewest` rows or more (shorter ones are left alone); `longest`: the most rows that one of them brings.  q and out as
// lab_attention_q8_any, q's rows on 16-byte boundaries.
LAB_EXPORT int lab_attention_q8_rows(void* out, int out_stride, const void* q, long long q_stride, const void* k, const void* v,
                                     const void* k_scale, const void* v_scale, const int* q_start, const int* kv_len, const int* pos0,
                                     const int* block_table, int max_blocks, int requests, int n_q, int n_kv, int page_size, int num_pages,
                                     int window, float scale, int fewest, int longest, cudaStream_t stream) {
  if (requests <= 0 || longest <= 0) return 0;
  if (n_kv < 1 || n_q < 1 || n_q % n_kv || max_blocks < 1 || num_pages < 1 || fewest < 1 ||
      !q8_pages_fit(page_size, (long long)num_pages * n_kv * page_size) || q_stride % 8 || (((uintptr_t)q) & 15) ||
      ((((uintptr_t)k) | ((uintptr_t)v)) & 15))
    return (int)cudaErrorInvalidValue;
  CUtensorMap mk, mv;
  int rc;
  const long long rows = (long long)num_pages * n_kv * page_size;
  if ((rc = q8_make_map<D>(&mk, k, rows, page_size))) return rc;
  if ((rc = q8_make_map<D>(&mv, v, rows, page_size))) return rc;
  Args a;
  a.out = (__nv_bfloat16*)out, a.out_stride = out_stride, a.q = (const __nv_bfloat16*)q, a.q_stride = q_stride;
  a.k_scale = (const uint8_t*)k_scale, a.v_scale = (const uint8_t*)v_scale;
  a.q_start = q_start, a.kv_len = kv_len, a.pos0 = pos0, a.block_table = block_table, a.max_blocks = max_blocks;
  a.n_q = n_q, a.n_kv = n_kv, a.page_size = page_size, a.num_pages = num_pages, a.window = window, a.fewest = fewest;
  a.scale_log2 = scale * LOG2E;
  static LabShared granted;
  cudaError_t e = lab_allow_shared(granted, (const void*)attention_q8_rows_kernel, SMEM);
  if (e != cudaSuccess) return (int)e;
  const long long tiles = ((long long)longest * (n_q / n_kv) + GROUPS * ROWS - 1) / (GROUPS * ROWS);
  return (int)lab_launch(attention_q8_rows_kernel, dim3(n_kv, (unsigned)tiles, requests), dim3(THREADS), (size_t)SMEM, stream, mk, mv, a);
}
