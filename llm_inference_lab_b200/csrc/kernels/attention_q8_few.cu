// Attention of few rows a request over the paged 8-bit cache (quant8.cuh) on the 5th-generation tensor cores, for heads of 64
// and 128 (-DLAB_HEAD_DIM) and pages of 8 to 128 tokens: single tokens, and the short portions that drafted tokens make.
//
// The rows of a request and kv head (its tokens times the query heads that share the kv head) are the short side of both
// products, N of them, a multiple of 16, and the keys the long one, so that the codes go to the tensor cores as TMA brings them
// and nothing is converted:
//   S^T [128 keys, N]  = K [128, D] Q^T                     kind::f8f6f4, K as cached, a row of 8-bit codes a key
//   P^T                = exp(S^T scaled, masked)            a thread a key
//   O^T [D, N]        += V^T [D, 128] P^T                   V as cached: the A operand, M-major
// q and p are cut into two codes each whose sum they are (quant8_tc.cuh), two products instead of one: q, after a power of
// two per row, is then exact but for parts below 2^-18 of the row's largest, and p good to 2^-8 at worst, twice as good as a
// bfloat16 on average.  The row scales being powers of two, a key's is a factor of its thread's scores and a value's an
// addend of the exponent: p' = 2^(s + e_v - M) with M the largest exponent of the TILE, per row.  A tile's p' then reach from
// 256 down to 2^-10, whatever earlier tiles held, so that a long tail behind one dominant key keeps its weight; the tile's O^T is
// read from tensor memory and added to the sums in registers with 2^(M - R), R the running reference.  A tile's sum of p
// without e_v is kept a thread for its own keys, and added over the threads once at the end.  (It is p' 2^-e_v: where a
// tile's values are rows of scales up to 2^90 apart and below 2^80, every weight down to 2^-44 of the largest is in it.)
//
// Warp 0 loads (TMA, a page a lane), warp 1 issues the products and owns tensor memory, warps 2-5 (128 threads) do the rest.
// The scores of tile j + 1 are formed beside the softmax of tile j, and O^T of tile j - 1 beside it too.  The keys are split
// over CTAs where there are fewer than the GPU holds, and merged inside a cluster of up to eight or by a second kernel.  Every wait
// is bounded.
//
// Memory bounds the loop (28 + 4 heads of 128, 32 requests of 4,096 keys: 29.3 us, 4.4 TB/s of keys and values, three CTAs a
// multiprocessor with a tile of 32 KB each every 3,000 to 4,000 cycles); what is above the bytes is the start, until the queries'
// codes are there, and the merge: most of a short call (14 + 2 heads of 64, 8 requests of 530 keys: 6.4 us; 16 requests of five
// drafted tokens over 1,700 keys, 12 + 2 heads of 128: 13.5 us).
#include "quant8_tc.cuh"

#ifndef LAB_HEAD_DIM
#error "build with -DLAB_HEAD_DIM=64 or 128"
#endif

namespace {

constexpr int D = LAB_HEAD_DIM;
using Tile = Q8Tile<D>;
constexpr int KEYS = Tile::KEYS;
constexpr int THREADS = 192;
constexpr int STAGES = D == 64 ? 4 : 2;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float FROM_CODES = 0.00390625f;      // p' is formed 2^8 times too large

template <int N> struct Layout {
  static constexpr int OFF_Q = 0;                                 // high, then low codes: [N, D] swizzled as the keys
  static constexpr int OFF_P = OFF_Q + 2 * N * D;                 // high, then low codes: slabs of 16 rows, [128 keys][16]
  static constexpr int OFF_K = OFF_P + 2 * N * KEYS;
  static constexpr int OFF_V = OFF_K + STAGES * Tile::BYTES;
  static constexpr int OFF_RED = OFF_V + STAGES * Tile::BYTES;    // [2][N][4] the warps' largest exponents of a tile
  static constexpr int OFF_ROW = OFF_RED + 2 * N * 16;            // per row: factor, last and first visible key
  static constexpr int OFF_WARP = OFF_ROW + 3 * N * 4;            // per warp: base, rescale, and two of the tile's factor
  static constexpr int OFF_BAR = OFF_WARP + 4 * 4 * N * 4;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;               // (1024: alignment)
  static constexpr int TM_S = 0, TM_O = 2 * N;
  static constexpr int TMEM = N <= 16 ? 64 : N <= 32 ? 128 : 256;
  static_assert(OFF_K % 1024 == 0 && (N * D) % 1024 == 0, "tiles begin where their swizzle does");
  static_assert(3 * N <= TMEM, "tensor memory holds two S and one O");
};

struct Barriers {
  uint64_t q_full, k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[2], s_empty[2], p_full, o_full;
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
  int tokens, max_blocks, n_q, n_kv, page_size, num_pages, window, most_rows, longest, splits, cluster, alone;
  bool by_request;      // the splits' results: `longest` places a request, else one a row of the batch
  float scale_log2;
  float *part_acc, *part_ml;
};

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void ld_cluster(uint32_t addr, float (&v)[2]) {
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ld_cluster(uint32_t addr, float (&v)[4]) {
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
}

// Sums of M rows' values (16 or 32) over a warp: lanes halve the rows between them, 16 exchanges for 16 rows and 31 for 32, five a
// row otherwise (16 requests of five drafted tokens: 13.4 us, 13.9).  Lane i gets row i * M / 32.
template <int M> __device__ __forceinline__ float warp_row_sums(const float* v, int lane) {
  float x[M];
#pragma unroll
  for (int i = 0; i < M; ++i) x[i] = v[i];
  int o = 16;
#pragma unroll
  for (int half = M / 2; half > 0; half /= 2, o /= 2) {
    const bool upper = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float give = upper ? x[i] : x[i + half], keep = upper ? x[i + half] : x[i];
      x[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
#pragma unroll
  for (int rest = 16 / M; rest > 0; rest /= 2) x[0] += __shfl_xor_sync(0xffffffffu, x[0], rest);
  return x[0];
}

template <int N>
__global__ void __launch_bounds__(THREADS, N <= 16 ? 3 : N <= 32 ? 2 : 1) attention_q8_few_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                   const __grid_constant__ CUtensorMap map_v, const Args a) {
  using L = Layout<N>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  Barriers* bar = reinterpret_cast<Barriers*>(smem + L::OFF_BAR);
  volatile int* abort_flag = &bar->abort_flag;
  pdl_trigger();
  // Until pdl_wait() below only the step's metadata is read (no kernel of the step writes it).
  const int b = blockIdx.z, split = blockIdx.x, group = a.n_q / a.n_kv;
  const int qs = a.q_start[b], ql = a.q_start[b + 1] - qs;
  const int tiles_of_rows = gridDim.y / a.n_kv, kvh = blockIdx.y / tiles_of_rows;
  const int r0 = (blockIdx.y - kvh * tiles_of_rows) * N;       // first row: row r is token r / group, head r % group
  const bool within = qs >= 0 && qs <= a.tokens - ql && ql <= a.longest;      // what the host has been told
  if (ql > a.most_rows || r0 >= ql * group || !within) {
    if ((ql <= a.most_rows || a.alone) && !within && r0 == 0 && threadIdx.x == 0) lab_set_error(LAB_ERR_ROW_RANGE);
    pdl_wait();  // this kernel ends only after the one before it: what follows may count on both
    return;
  }
  const int n_rows = min(N, ql * group - r0);
  const int p0 = a.pos0[b], kvl = a.kv_len[b];
  const int* bt = a.block_table + (size_t)b * a.max_blocks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pos_lo = p0 + r0 / group, pos_hi = p0 + (r0 + n_rows - 1) / group;
  const int last = min(min(pos_hi, kvl - 1), a.max_blocks * a.page_size - 1);      // last and first key that any row sees
  const int first = lab_first_key(pos_lo, a.window);
  const int t_first = first / KEYS, all_tiles = last >= first ? last / KEYS - t_first + 1 : 0;
  const int each = all_tiles / a.splits, more = all_tiles - each * a.splits;      // tiles of a split, and splits with one more
  const int t_lo = t_first + split * each + min(split, more), n_tiles = each + (split < more ? 1 : 0);
  const int page_shift = __ffs(a.page_size) - 1;

  if (threadIdx.x == 0) {
    mbar_init(&bar->q_full, 4);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&bar->k_full[s], 1);
      mbar_init(&bar->k_empty[s], 1);
      mbar_init(&bar->v_full[s], 1);
      mbar_init(&bar->v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->s_empty[i], 4);
    }
    mbar_init(&bar->p_full, 4);
    mbar_init(&bar->o_full, 1);
    bar->abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 0 && lane < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &map_k : &map_v) : "memory");
  if (warp == 1) tmem_alloc(&bar->tmem_slot, L::TMEM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem_base = bar->tmem_slot, smem_base = smem_u32(smem);
  // the pool's row of key j (all its heads' rows of a page lie one after the other), -1 if there is none to read
  auto row_of = [&](int j) -> long long {
    if (j < first || j > last) return -1;
    const int page = bt[j >> page_shift];
    return page < 0 || page >= a.num_pages ? -1 : (((long long)page * a.n_kv + kvh) << page_shift) + (j & (a.page_size - 1));
  };

  if (warp == 0) {
    // ---------------- loader: a page a lane ----------------
    const int pages_per_tile = KEYS >> page_shift, page_bytes = D << page_shift;
    // the pool's row of this lane's page in tile j, -1: not fetched (its keys are masked, its values set to zero)
    auto page_row = [&](int j) -> int {
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
      next = page_row(j + 1);      // looked up beside this tile's copies
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, row >= 0)) * page_bytes;
      // keys first: their place is free as soon as the scores are formed, the values' only after the softmax
      if (!__all_sync(0xffffffffu, mbar_wait(&bar->k_empty[s], ph ^ 1, abort_flag))) break;
      if (lane == 0) mbar_expect_tx(&bar->k_full[s], bytes);
      __syncwarp();
      if (row >= 0) tma_load_2d(smem_base + L::OFF_K + s * Tile::BYTES + lane * page_bytes, &map_k, &bar->k_full[s], 0, row);
      asked = 2 * j + 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&bar->v_empty[s], ph ^ 1, abort_flag))) break;
      if (lane == 0) mbar_expect_tx(&bar->v_full[s], bytes);
      __syncwarp();
      if (row >= 0) tma_load_2d(smem_base + L::OFF_V + s * Tile::BYTES + lane * page_bytes, &map_v, &bar->v_full[s], 0, row);
      asked = 2 * j + 2;
    }
    if (asked < 2 * n_tiles) {      // a wait has run out: the copies that were asked for land before the CTA ends
      volatile int never = 0;
      for (int i = max(0, asked - 2 * STAGES); i < asked; ++i) {
        const int j = i / 2, s = j % STAGES;
        mbar_wait(i & 1 ? &bar->v_full[s] : &bar->k_full[s], (j / STAGES) & 1, &never, 100000000ull);
      }
    }
  } else if (warp == 1) {
    // ---------------- products ----------------
    constexpr uint32_t idesc_s = q8_instr(KEYS, N, false, false), idesc_o = q8_instr(D, N, true, true);
    auto wait_all = [&](uint64_t* m, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(m, parity, abort_flag)); };
    const uint64_t q_high = q8_desc(smem_base + L::OFF_Q, 16, Tile::GROUP, Tile::LAYOUT),
                   q_low = q8_desc(smem_base + L::OFF_Q + N * D, 16, Tile::GROUP, Tile::LAYOUT);
    // p: a slab of 16 rows holds 16 bytes a key, 8 keys lie 128 bytes apart, the next slab 128 keys on
    const uint64_t p_high = q8_desc(smem_base + L::OFF_P, 128, KEYS * 16, 0), p_low = q8_desc(smem_base + L::OFF_P + N * KEYS, 128, KEYS * 16, 0);
    auto issue_s = [&](int j) -> bool {
      const int s = j % STAGES, sb = j & 1;
      if (!wait_all(&bar->k_full[s], (j / STAGES) & 1) || !wait_all(&bar->s_empty[sb], ((j >> 1) & 1) ^ 1)) return false;
      tc_fence_after();
      const uint64_t kd = q8_desc(smem_base + L::OFF_K + s * Tile::BYTES, 16, Tile::GROUP, Tile::LAYOUT);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) umma_q8(tmem_base + L::TM_S + sb * N, kd + 2 * k, q_high + 2 * k, idesc_s, k > 0);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) umma_q8(tmem_base + L::TM_S + sb * N, kd + 2 * k, q_low + 2 * k, idesc_s, 1);
      umma_commit(&bar->s_full[sb]);
      umma_commit(&bar->k_empty[s]);
      return true;
    };
    bool ok = n_tiles > 0 && wait_all(&bar->q_full, 0) && issue_s(0);
    for (int j = 0; j < n_tiles && ok; ++j) {
      if (j + 1 < n_tiles && !issue_s(j + 1)) break;
      const int s = j % STAGES;
      if (!wait_all(&bar->v_full[s], (j / STAGES) & 1) || !wait_all(&bar->p_full, j & 1)) break;
      tc_fence_after();
      const uint64_t vd = q8_desc(smem_base + L::OFF_V + s * Tile::BYTES, 16, Tile::GROUP, Tile::LAYOUT);
#pragma unroll
      for (int k = 0; k < KEYS / 32; ++k)
        umma_q8(tmem_base + L::TM_O, vd + (uint64_t)(k * 32 * D / 16), p_high + (uint64_t)(k * 32), idesc_o, k > 0);
#pragma unroll
      for (int k = 0; k < KEYS / 32; ++k)
        umma_q8(tmem_base + L::TM_O, vd + (uint64_t)(k * 32 * D / 16), p_low + (uint64_t)(k * 32), idesc_o, 1);
      umma_commit(&bar->o_full);
      umma_commit(&bar->v_empty[s]);
    }
  } else {
    // ---------------- a thread a key, and for O^T a thread an entry of the head ----------------
    const int quarter = warp & 3, w = warp - 2;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    float* factor = reinterpret_cast<float*>(smem + L::OFF_ROW);
    int* row_last = reinterpret_cast<int*>(factor + N);
    int* row_first = row_last + N;
    float* base_w = reinterpret_cast<float*>(smem + L::OFF_WARP) + w * 4 * N;      // [N] base, [N] rescale, [2][N] share
    float *rescale_w = base_w + N, *share_w = base_w + 2 * N;
    // the first key's bytes are on their way beside the queries
    const int mine = quarter * 32 + lane;
    long long row = n_tiles > 0 ? row_of(t_lo * KEYS + mine) : -1;
    uint32_t kb = row >= 0 ? a.k_scale[row] : 127, vb = row >= 0 ? a.v_scale[row] : 127;
    // q: scaled by a power of two per row, in two codes.  Eight lanes a row, sixteen rows a pass, all loads in flight together; the
    // passes are one piece of code, as it runs once and its instructions are fetched while it does (16 requests of five drafted
    // tokens: 14.0 us, 15.4 with a row a warp and turn, unrolled, whose codes alone took 8,600 cycles).
    constexpr int PASSES = N / 16, EACH = D / 8;      // numbers of a row a lane
    const int in_pass = (w * 32 + lane) >> 3, sub = lane & 7;
    uint32_t x[PASSES][EACH / 2];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int n = 16 * p + in_pass, r = r0 + n, token = r / group, head = kvh * group + r - token * group;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(a.q + (size_t)(qs + token) * a.q_stride + (size_t)head * D + sub * EACH);
#pragma unroll
      for (int e = 0; e < EACH / 2; ++e) x[p][e] = n < n_rows ? src[e] : 0u;
      if (sub == 0) {
        const int pos = p0 + token;
        row_last[n] = n < n_rows ? min(pos, last) : -1;
        row_first[n] = lab_first_key(pos, a.window);
      }
    }
#pragma unroll 1
    for (int p = 0; p < PASSES; ++p) {
      const int n = 16 * p + in_pass;
      uint32_t top = 0;      // of the numbers' upper 16 bits
#pragma unroll
      for (int e = 0; e < EACH / 2; ++e) top = max(top, max(x[0][e] & 0x7fff0000u, (x[0][e] << 16) & 0x7fff0000u));
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int byte = q8_byte(top);
      const float inverse = q8_inverse(min(byte, 253));
      uint32_t high[EACH / 4], low[EACH / 4];
#pragma unroll
      for (int e = 0; e < EACH / 4; ++e) {
        const uint32_t u = byte == Q8_NAN_BYTE ? 0u : x[0][2 * e], v = byte == Q8_NAN_BYTE ? 0u : x[0][2 * e + 1];
        const float f[4] = {__uint_as_float(u << 16) * inverse, __uint_as_float(u & 0xffff0000u) * inverse, __uint_as_float(v << 16) * inverse,
                            __uint_as_float(v & 0xffff0000u) * inverse};
        q8_split4(f, high[e], low[e]);
      }
      uint8_t* to = smem + L::OFF_Q + Tile::piece_at(n, sub * EACH >> 4) + (sub * EACH & 15);
      if constexpr (D == 128) {
        *reinterpret_cast<uint4*>(to) = make_uint4(high[0], high[1], high[2], high[3]);
        *reinterpret_cast<uint4*>(to + N * D) = make_uint4(low[0], low[1], low[2], low[3]);
      } else {
        *reinterpret_cast<uint2*>(to) = make_uint2(high[0], high[1]);
        *reinterpret_cast<uint2*>(to + N * D) = make_uint2(low[0], low[1]);
      }
      if (sub == 0) factor[n] = n < n_rows ? a.scale_log2 * q8_scale(byte) : 0.f;
#pragma unroll
      for (int i = 0; i + 1 < PASSES; ++i)
#pragma unroll
        for (int e = 0; e < EACH / 2; ++e) x[i][e] = x[i + 1][e];
    }
    proxy_fence();
    asm volatile("bar.sync 2, 128;" ::: "memory");      // the rows' numbers
    if (lane == 0) mbar_arrive(&bar->q_full);

    float acc[N], l[N], ref = -INFINITY, ref2 = -INFINITY;      // references of rows lane and lane + 32
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] = l[n] = 0.f;
    auto add_o = [&](int j) -> bool {      // O^T of tile j into the sums, by the tile's factors
      if (!__all_sync(0xffffffffu, mbar_wait(&bar->o_full, j & 1, abort_flag))) return false;
      tc_fence_after();
      const float* share = share_w + (j & 1) * N;
#pragma unroll
      for (int n0 = 0; n0 < N; n0 += 16) {
        uint32_t r[16];
        tmem_ld16_issue(lane_addr + L::TM_O + n0, r);
        tmem_wait();
#pragma unroll
        for (int n = 0; n < 16; n += 4) {
          const float4 f = load4(share + n0 + n);
          acc[n0 + n] = fmaf(__uint_as_float(r[n]), f.x, acc[n0 + n]);
          acc[n0 + n + 1] = fmaf(__uint_as_float(r[n + 1]), f.y, acc[n0 + n + 1]);
          acc[n0 + n + 2] = fmaf(__uint_as_float(r[n + 2]), f.z, acc[n0 + n + 2]);
          acc[n0 + n + 3] = fmaf(__uint_as_float(r[n + 3]), f.w, acc[n0 + n + 3]);
        }
      }
      return true;
    };
    // Where a wait has run out the four warps still walk to the end, so that they keep meeting at their barriers (no further
    // wait lasts: each sees that one has given up); nothing is written then.
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      const int key = (t_lo + j) * KEYS + mine, key0 = (t_lo + j) * KEYS;
      const bool held = row >= 0;
      const bool unit = held && vb == 127;
      float vexp = (float)((int)vb - 127), v_inv = __uint_as_float((uint32_t)(254 - min(vb, 253u)) << 23) * FROM_CODES;
      const float ks = vb == Q8_NAN_BYTE ? q8_scale(Q8_NAN_BYTE) : q8_scale(kb);      // a value that is no number, as a score that is none
      if (j + 1 < n_tiles) {      // the next key's bytes arrive beside this tile
        row = row_of(key + KEYS);
        kb = row >= 0 ? a.k_scale[row] : 127, vb = row >= 0 ? a.v_scale[row] : 127;
      }
      if (__any_sync(0xffffffffu, unit)) {
        // A scale of one may be that of a value of zeros, which must not set the tile's largest p' (behind a first token with
        // all the weight and nothing to say the others' p' would be below the smallest code).  Any other power gives the same
        // sums: it takes one 2^60 below the largest of the warp's other values, so that a key of 2^60 times the others' weight
        // leaves them theirs, and that its own weight reaches the sum down to 2^-60 of the largest.
        ok &= __all_sync(0xffffffffu, mbar_wait(&bar->v_full[j % STAGES], (j / STAGES) & 1, abort_flag));
        uint32_t any = unit ? 0u : 1u;
        if (unit) {
          const uint4* z = reinterpret_cast<const uint4*>(smem + L::OFF_V + (j % STAGES) * Tile::BYTES + mine * D);
#pragma unroll
          for (int c = 0; c < D / 16; ++c) any |= z[c].x | z[c].y | z[c].z | z[c].w;
        }
        const bool nothing = (any & 0x7f7f7f7fu) == 0;
        const float others = warp_max_number(held && !nothing && vexp < 128.f ? vexp : -INFINITY);      // (128: a value that is no number)
        if (nothing) {
          vexp = fmaxf((others == -INFINITY ? 0.f : others) - 60.f, (float)Q8_LEAST_POWER);
          v_inv = __uint_as_float((uint32_t)(127 - (int)vexp) << 23) * FROM_CODES;
        }
      }
      const int sb = j & 1;
      ok &= __all_sync(0xffffffffu, mbar_wait(&bar->s_full[sb], (j >> 1) & 1, abort_flag));
      tc_fence_after();
      float t[N];
#pragma unroll
      for (int n0 = 0; n0 < N; n0 += 16) tmem_ld16_issue(lane_addr + L::TM_S + sb * N + n0, reinterpret_cast<uint32_t*>(t) + n0);
      tmem_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->s_empty[sb]);
      const bool whole = key0 >= lab_first_key(pos_hi, a.window) && key0 + KEYS - 1 <= min(pos_lo, last);
#pragma unroll
      for (int n = 0; n < N; n += 4) {
        const float4 f = load4(factor + n);
        t[n] = fmaf(t[n] * ks, f.x, vexp);
        t[n + 1] = fmaf(t[n + 1] * ks, f.y, vexp);
        t[n + 2] = fmaf(t[n + 2] * ks, f.z, vexp);
        t[n + 3] = fmaf(t[n + 3] * ks, f.w, vexp);
      }
      if (!whole || !held) {
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (!held || key > row_last[n] || key < row_first[n]) t[n] = -INFINITY;
      }
      // the tile's largest exponent per row: over the warp, then over the four warps
      float* red = reinterpret_cast<float*>(smem + L::OFF_RED) + (j & 1) * N * 4;
#pragma unroll
      for (int n0 = 0; n0 < N; n0 += 32) {
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < 32 && n0 + n < N; ++n) {
          const float m = warp_max_number(t[n0 + n]);
          if (lane == n) top = m;
        }
        if (n0 + lane < N) red[(n0 + lane) * 4 + w] = top;
      }
      asm volatile("bar.sync 2, 128;" ::: "memory");
      bool grew = false;
#pragma unroll
      for (int n0 = 0; n0 < N; n0 += 32) {
        if (n0 + lane < N) {
          const float4 m4 = load4(red + (n0 + lane) * 4);
          const float m = fmaxf(fmaxf(m4.x, m4.y), fmaxf(m4.z, m4.w));
          float& r = n0 == 0 ? ref : ref2;
          const float r_new = fmaxf(r, m);
          grew |= r_new > r && r != -INFINITY;
          base_w[n0 + lane] = m == -INFINITY ? 0.f : m - 8.f;      // p' up to 2^8
          rescale_w[n0 + lane] = r == r_new ? 1.f : fast_exp2(r - r_new);
          share_w[(j & 1) * N + n0 + lane] = m == -INFINITY ? 0.f : fast_exp2(m - r_new);
          r = r_new;
        }
      }
      grew = __any_sync(0xffffffffu, grew);
      __syncwarp();
      // p', its two codes, and its share of the sum; an earlier tile's product is done reading the codes once its O^T is
#pragma unroll
      for (int n = 0; n < N; n += 4) {
        const float4 m = load4(base_w + n);
        t[n] = fast_exp2(t[n] - m.x);
        t[n + 1] = fast_exp2(t[n + 1] - m.y);
        t[n + 2] = fast_exp2(t[n + 2] - m.z);
        t[n + 3] = fast_exp2(t[n + 3] - m.w);
      }
      if (j > 0) ok &= add_o(j - 1);
      if (grew) {
#pragma unroll
        for (int n = 0; n < N; n += 4) {
          const float4 f = load4(rescale_w + n);
          acc[n] *= f.x, acc[n + 1] *= f.y, acc[n + 2] *= f.z, acc[n + 3] *= f.w;
          l[n] *= f.x, l[n + 1] *= f.y, l[n + 2] *= f.z, l[n + 3] *= f.w;
        }
      }
#pragma unroll
      for (int n = 0; n < N; n += 4) {
        const float4 f = load4(share_w + (j & 1) * N + n);
        l[n] = fmaf(t[n] * v_inv, f.x, l[n]);
        l[n + 1] = fmaf(t[n + 1] * v_inv, f.y, l[n + 1]);
        l[n + 2] = fmaf(t[n + 2] * v_inv, f.z, l[n + 2]);
        l[n + 3] = fmaf(t[n + 3] * v_inv, f.w, l[n + 3]);
      }
#pragma unroll
      for (int n0 = 0; n0 < N; n0 += 16) {
        uint32_t high[4], low[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x[4] = {t[n0 + 4 * e], t[n0 + 4 * e + 1], t[n0 + 4 * e + 2], t[n0 + 4 * e + 3]};
          q8_split4(x, high[e], low[e]);
        }
        uint8_t* to = smem + L::OFF_P + n0 * KEYS + mine * 16;
        *reinterpret_cast<uint4*>(to) = make_uint4(high[0], high[1], high[2], high[3]);
        *reinterpret_cast<uint4*>(to + N * KEYS) = make_uint4(low[0], low[1], low[2], low[3]);
      }
      if (__any_sync(0xffffffffu, !held)) {
        // a key that is not there: its place holds what an earlier owner left, and 0 times a code that is no number would be none
        ok &= __all_sync(0xffffffffu, mbar_wait(&bar->v_full[j % STAGES], (j / STAGES) & 1, abort_flag));
        if (!held) {
          uint4* z = reinterpret_cast<uint4*>(smem + L::OFF_V + (j % STAGES) * Tile::BYTES + mine * D);
#pragma unroll
          for (int c = 0; c < D / 16; ++c) z[c] = make_uint4(0, 0, 0, 0);
        }
      }
      proxy_fence();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->p_full);
    }
    if (n_tiles > 0) ok &= add_o(n_tiles - 1);
    // the rows' sums over the 128 threads, and the result
    float* sums = reinterpret_cast<float*>(smem + L::OFF_RED);      // [N][4]
    asm volatile("bar.sync 2, 128;" ::: "memory");      // (the last tile's exponents have been read)
#pragma unroll
    for (int n0 = 0; n0 < N; n0 += 32) {
      constexpr int LAST = N % 32 == 0 ? 32 : 16;
      if (n0 + 32 <= N) {
        sums[(n0 + lane) * 4 + w] = warp_row_sums<32>(l + n0, lane);
      } else {
        const float own = warp_row_sums<LAST>(l + n0, lane);
        if (lane % (32 / LAST) == 0) sums[(n0 + lane * LAST / 32) * 4 + w] = own;
      }
      if (n0 + lane < N) base_w[n0 + lane] = n0 == 0 ? ref : ref2;
    }
    asm volatile("bar.sync 2, 128;" ::: "memory");
    const int dim = D == 128 ? mine : quarter * 16 + lane;      // (64 rows of an accumulator: 16 lanes a quarter)
    float* own = reinterpret_cast<float*>(smem + L::OFF_K);     // in a cluster: [N][D], then [N] references and [N] sums
    if (a.cluster && w == 0) {
      for (int n = lane; n < N; n += 32) {
        const float4 s4 = load4(sums + n * 4);
        own[N * D + n] = ok ? base_w[n] : -INFINITY;
        own[N * D + N + n] = ok ? (s4.x + s4.y) + (s4.z + s4.w) : 0.f;
      }
    }
    if (ok && (D == 128 || lane < 16)) {
      if (a.cluster) {
#pragma unroll
        for (int n = 0; n < N; ++n) own[n * D + dim] = acc[n];
      } else {
        int token = r0 / group, head = r0 - token * group;      // of the row, counted on
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (n >= n_rows) break;
          const float4 s4 = load4(sums + n * 4);
          const float sum = (s4.x + s4.y) + (s4.z + s4.w), num = acc[n] * FROM_CODES;
          if (a.splits == 1) {
            a.out[(size_t)(qs + token) * a.out_stride + (size_t)(kvh * group + head) * D + dim] = __float2bfloat16_rn(sum == 0.f ? 0.f : num / sum);
          } else {
            const size_t slot = ((size_t)((a.by_request ? b * a.longest : qs) + token) * a.n_q + kvh * group + head) * a.splits + split;
            a.part_acc[slot * D + dim] = num;
            if (dim == 0) a.part_ml[slot * 2] = base_w[n], a.part_ml[slot * 2 + 1] = sum;
          }
          if (++head == group) head = 0, ++token;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::TMEM);
  }
  if (a.cluster) {
    // The splits of these rows are the cluster's CTAs: each merges every splits-th row out of the others' shared memory, a warp a row.
    cluster_sync();
    const uint32_t theirs = smem_base + L::OFF_K, at = map_to_rank(theirs, lane < a.splits ? lane : 0);
    for (int n = split + warp * a.splits; n < n_rows; n += THREADS / 32 * a.splits) {
      // lane i: split i's reference and sum
      const float m = lane < a.splits ? ld_cluster_f32(at + (N * D + n) * 4) : -INFINITY, l = lane < a.splits ? ld_cluster_f32(at + (N * D + N + n) * 4) : 0.f;
      const float big = warp_max_number(m), f = m == -INFINITY ? 0.f : fast_exp2(m - big);
      const float den = warp_sum(f * l);      // (0 times a NaN is one: scores that are all none stay visible)
      constexpr int EACH = D / 32;
      float v[8][EACH], num[EACH];
#pragma unroll
      for (int i = 0; i < 8; ++i) ld_cluster(map_to_rank(theirs, i < a.splits ? i : 0) + (n * D + lane * EACH) * 4, v[i]);
#pragma unroll
      for (int e = 0; e < EACH; ++e) num[e] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float fi = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
        for (int e = 0; e < EACH; ++e) num[e] = i < a.splits ? fmaf(fi, v[i][e], num[e]) : num[e];
      }
      const int r = r0 + n, token = r / group, head = kvh * group + r - token * group;
      __nv_bfloat16* to = a.out + (size_t)(qs + token) * a.out_stride + (size_t)head * D + lane * EACH;
      const float inverse = den == 0.f ? 0.f : FROM_CODES / den;
#pragma unroll
      for (int e = 0; e < EACH; ++e) to[e] = __float2bfloat16_rn(num[e] * inverse);
    }
    cluster_sync();      // nobody's shared memory goes before the others have read it
  }
}

// The splits of a row and query head put together: a block each, a thread an entry, PARTS of them over the splits.
constexpr int MERGE_PARTS = 1024 / 128;
template <int PARTS>
__global__ void __launch_bounds__(PARTS* D) attention_q8_merge_kernel(const Args a) {
  __shared__ float num_s[PARTS][D], m_s[PARTS], den_s[PARTS];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.z, head = blockIdx.y, dim = threadIdx.x % D, part = threadIdx.x / D;
  const int qs = a.q_start[b], ql = a.q_start[b + 1] - qs, token = blockIdx.x;
  if (ql > a.most_rows || token >= ql || qs < 0 || qs > a.tokens - ql || ql > a.longest) return;
  const size_t slot = ((size_t)((a.by_request ? b * a.longest : qs) + token) * a.n_q + head) * a.splits;
  const int each = (a.splits + PARTS - 1) / PARTS, end = min(a.splits, (part + 1) * each);
  float big = -INFINITY, num = 0.f, den = 0.f;
  for (int s0 = part * each; s0 < end; s0 += 8) {      // eight splits' loads in flight, added in their order
    float acc[8], m[8], l[8], most = big;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = s0 + i < end;
      m[i] = in ? a.part_ml[(slot + s0 + i) * 2] : -INFINITY;
      l[i] = in ? a.part_ml[(slot + s0 + i) * 2 + 1] : 0.f;
      acc[i] = in ? a.part_acc[(slot + s0 + i) * D + dim] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, m[i]);
    const float f0 = big == most ? 1.f : fast_exp2(big - most);
    num *= f0, den *= f0, big = most;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = m[i] == -INFINITY ? 0.f : fast_exp2(m[i] - big);
      num = fmaf(f, acc[i], num);
      den = fmaf(f, l[i], den);      // (0 times a NaN is one: scores that are all none stay visible)
    }
  }
  if constexpr (PARTS > 1) {
    num_s[part][dim] = num;
    if (dim == 0) m_s[part] = big, den_s[part] = den;
    __syncthreads();
    if (part > 0) return;
    big = -INFINITY, num = 0.f, den = 0.f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) big = fmaxf(big, m_s[i]);
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const float f = m_s[i] == -INFINITY ? 0.f : fast_exp2(m_s[i] - big);
      num = fmaf(f, num_s[i][dim], num);
      den = fmaf(f, den_s[i], den);
    }
  }
  a.out[(size_t)(qs + token) * a.out_stride + (size_t)head * D + dim] = __float2bfloat16_rn(den == 0.f ? 0.f : num / den);
}

template <int N>
int launch_few(const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, dim3 grid, cudaStream_t stream) {
  static LabShared granted;
  cudaError_t e = lab_allow_shared(granted, (const void*)attention_q8_few_kernel<N>, Layout<N>::SMEM);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Layout<N>::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (a.cluster) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = a.splits;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (g_lab_pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return (int)cudaLaunchKernelEx(&cfg, attention_q8_few_kernel<N>, mk, mv, a);
}

template <int N>
int clusters_of(int size) {
  static LabShared granted;
  if (lab_allow_shared(granted, (const void*)attention_q8_few_kernel<N>, Layout<N>::SMEM) != cudaSuccess) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Layout<N>::SMEM;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  return cudaOccupancyMaxActiveClusters(&n, (const void*)attention_q8_few_kernel<N>, &cfg) == cudaSuccess ? n : -1;
}

}  // namespace

// Clusters of `size` CTAs of a width that the current device holds at once, -1 where it does not say.
LAB_EXPORT int lab_attention_q8_few_clusters(int width, int size) {
  if (size < 1 || size > 8) return -1;
  return width == 16 ? clusters_of<16>(size) : width == 32 ? clusters_of<32>(size) : width == 48 ? clusters_of<48>(size) : -1;
}

// A call, as the host packs it.  q: `tokens` rows q_stride elements apart, out likewise; requests of up to most_rows rows (longer
// ones are left alone, and reported where no other call takes them: `alone`), `longest` the most that one of them brings; width: rows a
// CTA takes, 16, 32 or 48; splits of the keys, merged inside their cluster (`cluster`, up to eight) or by a second kernel through
// scratch: n_q * splits * (D + 2) floats for each of min(tokens, requests * longest) rows.
// window as lab_first_key takes it.
struct LabQ8Few {
  void* out;
  const void *q, *k, *v, *k_scale, *v_scale;
  const int *q_start, *kv_len, *pos0, *block_table;
  float* scratch;
  long long out_stride, q_stride;
  int tokens, max_blocks, requests, n_q, n_kv, page_size, num_pages, window, most_rows, longest, width, splits, cluster, alone;
  float scale;
};

LAB_EXPORT int lab_attention_q8_few(const LabQ8Few* c, cudaStream_t stream) {
  if (c->tokens <= 0 || c->requests <= 0 || c->longest <= 0) return 0;
  if (c->n_kv < 1 || c->n_q < 1 || c->n_q % c->n_kv || c->splits < 1 || c->max_blocks < 1 || c->longest > c->most_rows ||
      (c->cluster && (c->splits < 2 || c->splits > 8)) || (c->splits > 1 && !c->cluster && c->scratch == nullptr) ||
      !q8_pages_fit(c->page_size, (long long)c->num_pages * c->n_kv * c->page_size) || c->num_pages < 1 || c->q_stride % 2 ||
      c->requests > 65535 || c->n_q > 65535 || (((uintptr_t)c->q) & 3) || ((((uintptr_t)c->k) | ((uintptr_t)c->v)) & 15))
    return (int)cudaErrorInvalidValue;
  CUtensorMap mk, mv;
  int rc;
  const long long rows = (long long)c->num_pages * c->n_kv * c->page_size;
  if ((rc = q8_make_map<D>(&mk, c->k, rows, c->page_size))) return rc;
  if ((rc = q8_make_map<D>(&mv, c->v, rows, c->page_size))) return rc;
  Args a;
  a.out = (__nv_bfloat16*)c->out, a.out_stride = c->out_stride, a.q = (const __nv_bfloat16*)c->q, a.q_stride = c->q_stride;
  a.k_scale = (const uint8_t*)c->k_scale, a.v_scale = (const uint8_t*)c->v_scale;
  a.q_start = c->q_start, a.kv_len = c->kv_len, a.pos0 = c->pos0, a.block_table = c->block_table, a.max_blocks = c->max_blocks;
  a.n_q = c->n_q, a.n_kv = c->n_kv, a.page_size = c->page_size, a.num_pages = c->num_pages, a.window = c->window;
  a.most_rows = c->most_rows, a.splits = c->splits, a.cluster = c->cluster, a.alone = c->alone, a.scale_log2 = c->scale * LOG2E;
  const bool second = c->splits > 1 && !c->cluster;
  a.tokens = c->tokens, a.longest = c->longest;
  const long long places = (long long)c->requests * c->longest;
  a.by_request = places < c->tokens;      // (a long portion beside a few single tokens takes no place)
  a.part_acc = c->scratch, a.part_ml = second ? c->scratch + (size_t)(a.by_request ? places : c->tokens) * c->n_q * c->splits * D : nullptr;
  const int row_tiles = (c->longest * (c->n_q / c->n_kv) + c->width - 1) / c->width;
  if ((long long)c->n_kv * row_tiles > 65535) return (int)cudaErrorInvalidValue;
  const dim3 grid(c->splits, c->n_kv * row_tiles, c->requests);
  if (c->width == 16) rc = launch_few<16>(mk, mv, a, grid, stream);
  else if (c->width == 32) rc = launch_few<32>(mk, mv, a, grid, stream);
  else if (c->width == 48) rc = launch_few<48>(mk, mv, a, grid, stream);
  else rc = (int)cudaErrorInvalidValue;
  if (rc || !second) return rc;
  const dim3 heads(c->longest, c->n_q, c->requests);
  if (c->splits > 16) return (int)lab_launch(attention_q8_merge_kernel<MERGE_PARTS>, heads, dim3(MERGE_PARTS * D), 0, stream, a);
  return (int)lab_launch(attention_q8_merge_kernel<1>, heads, dim3(D), 0, stream, a);
}
