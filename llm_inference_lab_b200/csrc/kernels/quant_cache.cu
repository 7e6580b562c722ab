// A paged cache in 8 bits (quant8.cuh): keys rotated, keys and values rounded and written to their pages, and rows of such
// pages read back.
//
//   store   q' = q turned by its row's angles, rounded to the storage type; k' = k turned, v: to codes and a byte a row
//           (lo, hi) -> (lo c - hi s, hi c + lo s), elements i and i + rotary_dim / 2 of a head; c, s from the step's table
//   load    code * 2^(e - 127)
//
// A key's code is the one nearest to the exact k': the products of 8- or 24-bit numbers with the table's are formed in 64 bits,
// and one rounding leads from there to 8 bits (a product rounded to 32 bits, let alone to 16, before its code is chosen takes
// the neighbouring code now and then).  So the cache depends on the inputs alone, not on the order of anything.  Queries are turned in 32
// bits as everywhere (rowwise.cu): their result is rounded once.
//
// Both are bound by memory: a row's lanes hold it in registers between the one read and the one write, and the row's largest
// magnitude goes around its lanes by shuffles.
#include "quant8.cuh"

namespace {

constexpr int THREADS = 256, FEW_THREADS = 64, VEC_THREADS = 128;
constexpr int MOST_DIM = 256;

struct Store {
  const void* rows;          // [tokens, row_stride] of T, or [parts, tokens, width] floats
  long long row_stride;
  int parts;                 // 0: rows of T
  long long part_stride;
  const __nv_bfloat16* bias; // [width] or null (parts only)
  const float2* table;       // [tokens, rotary_dim / 2] (cos, sin), null with rotary_dim 0
  int rotary_dim;
  const int* slots;          // [tokens], negative: not stored
  void* q_out;               // [tokens, n_q * d] of T
  uint8_t *k, *v, *k_scale, *v_scale;
  int tokens, n_q, n_kv, d, page_size, num_pages;
};

// Where a row of the cache lies: its number among the pool's rows, or -1.
__device__ __forceinline__ long long pool_row(const Store& s, int token, int kv_head, bool reports) {
  const int slot = s.slots[token];
  if (slot < 0) return -1;
  const int page = slot / s.page_size;
  if (page >= s.num_pages) {
    if (reports) lab_set_error(LAB_ERR_PAGE_RANGE);
    return -1;
  }
  return ((long long)page * s.n_kv + kv_head) * s.page_size + (slot - page * s.page_size);
}

// N neighbouring numbers of a row.  PARTS: the parts are summed in 64 bits in their order, the bias added, and the sum rounded
// to 32 bits, as a product in one piece leaves it, and then to bfloat16, the type that the rows would have.
template <typename T, bool PARTS, int N>
__device__ __forceinline__ void take(const Store& s, int token, int col, float (&x)[N]) {
  if constexpr (PARTS) {
    const float* p = static_cast<const float*>(s.rows) + (size_t)token * s.row_stride + col;
    double sum[N];
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = 0.0;
    for (int s0 = 0; s0 < s.parts; s0 += 8) {      // eight loads in flight
      float f[8][N];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) f[i][j] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s0 + i < s.parts) {
          if constexpr (N == 2) {
            const float2 w = *reinterpret_cast<const float2*>(p + (s0 + i) * s.part_stride);
            f[i][0] = w.x, f[i][1] = w.y;
          } else {
            f[i][0] = p[(s0 + i) * s.part_stride];
          }
        }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] += f[i][j];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (s.bias) sum[j] += to_f32(s.bias[col + j]);
      x[j] = round_to<__nv_bfloat16>((float)sum[j]);
    }
  } else {
    const T* p = static_cast<const T*>(s.rows) + (size_t)token * s.row_stride + col;
    if constexpr (N == 8) {
      const float4 a = load4(p), b = load4(p + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = to_f32(p[j]);
    }
  }
}
// 16 bytes a load where the row's bytes allow it: bfloat16 rows, eight at a time.
template <>
__device__ __forceinline__ void take<__nv_bfloat16, false, 8>(const Store& s, int token, int col, float (&x)[8]) {
  const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(s.rows) + (size_t)token * s.row_stride + col);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
}

template <int N> __device__ __forceinline__ void put(__nv_bfloat16* to, const float (&x)[N]) {
  if constexpr (N == 8)
    *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  else
    *reinterpret_cast<uint32_t*>(to) = pack_bf16(x[0], x[1]);
}
template <int N> __device__ __forceinline__ void put(float* to, const float (&x)[N]) {
  if constexpr (N == 8) {
    store4(to, make_float4(x[0], x[1], x[2], x[3]));
    store4(to + 4, make_float4(x[4], x[5], x[6], x[7]));
  } else {
    *reinterpret_cast<float2*>(to) = make_float2(x[0], x[1]);
  }
}
template <int N> __device__ __forceinline__ void put_codes(uint8_t* to, const float (&x)[N], float inverse) {
  if constexpr (N == 8)
    *reinterpret_cast<uint2*>(to) = make_uint2(q8_encode4(x[0] * inverse, x[1] * inverse, x[2] * inverse, x[3] * inverse),
                                               q8_encode4(x[4] * inverse, x[5] * inverse, x[6] * inverse, x[7] * inverse));
  else
    *reinterpret_cast<uint16_t*>(to) = (uint16_t)q8_encode2(x[0] * inverse, x[1] * inverse);
}

// Whole heads rotated, d a power of two from 16 to 256 (128 for parts: a row's lanes are one warp's), everything on the boundaries
// of its vectors: d / (2 N) lanes a row, each with N elements of its first half and the N that they turn with.  N = 8 (16 bytes of
// bfloat16 a load) for rows; N = 2 for parts, whose steps have few rows: four times the lanes then share the sums.  Blocks of 128,
// ten a multiprocessor (2,048 tokens of 28 + 8 heads of 128: 11.1 to 11.7 us by what runs around it, 12.1 where that is 11.1 by blocks of
// 256, four of them; the loads' latency bounds it, 3.2 TB/s).
template <typename T, bool PARTS, int N>
__global__ void __launch_bounds__(PARTS ? FEW_THREADS : VEC_THREADS, PARTS ? 1 : 10) store_vec_kernel(const Store s) {
  pdl_trigger();
  pdl_wait();
  const int half = s.d / 2, lanes = half / N, shift = __ffs(lanes) - 1, heads = s.n_q + 2 * s.n_kv;
  const unsigned unit = blockIdx.x * blockDim.x + threadIdx.x, row = unit >> shift, rows = (unsigned)s.tokens * heads;      // (the host checks: below 2^31)
  if ((unit & ~31u) >> shift >= rows) return;      // the whole warp
  const bool there = row < rows;
  const int token = there ? (int)(row / heads) : s.tokens - 1, head = there ? (int)(row - token * heads) : heads - 1;
  const int at = (int)(unit & (lanes - 1)) * N;
  float lo[N], hi[N];
  take<T, PARTS, N>(s, token, head * s.d + at, lo);
  take<T, PARTS, N>(s, token, head * s.d + at + half, hi);
  float2 turn[N];
  if (head < s.n_q + s.n_kv) {
    const float4* t = reinterpret_cast<const float4*>(s.table + (size_t)token * half + at);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      const float4 f = t[j];
      turn[2 * j] = make_float2(f.x, f.y), turn[2 * j + 1] = make_float2(f.z, f.w);
    }
  }
  const bool stored = head >= s.n_q;
  if (head < s.n_q) {
#pragma unroll
    for (int j = 0; j < N; ++j) rope_rotate(lo[j], hi[j], turn[j].x, turn[j].y, lo[j], hi[j]);
    using O = T;
    O* to = static_cast<O*>(s.q_out) + (size_t)token * s.n_q * s.d + head * s.d + at;
    if (there) put<N>(to, lo), put<N>(to + half, hi);
  } else if (head < s.n_q + s.n_kv) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const double a = lo[j], b = hi[j], c = turn[j].x, n = turn[j].y;
      lo[j] = q8_to_odd(a * c - b * n);
      hi[j] = q8_to_odd(b * c + a * n);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) top = max(top, max(__float_as_uint(lo[j]) & 0x7fffffffu, __float_as_uint(hi[j]) & 0x7fffffffu));
  for (int o = lanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (!there || !stored) return;
  const bool is_v = head >= s.n_q + s.n_kv;
  const long long place = pool_row(s, token, head - s.n_q - (is_v ? s.n_kv : 0), at == 0);
  if (place < 0) return;
  const int byte = q8_byte(top);
  if (byte == Q8_NAN_BYTE) {
#pragma unroll
    for (int j = 0; j < N; ++j) lo[j] = hi[j] = 0.f;
  }
  const float inverse = byte == Q8_NAN_BYTE ? 0.f : q8_inverse(byte);
  uint8_t* to = (is_v ? s.v : s.k) + place * s.d + at;
  put_codes<N>(to, lo, inverse);
  put_codes<N>(to + half, hi, inverse);
  if (at == 0) (is_v ? s.v_scale : s.k_scale)[place] = (uint8_t)byte;
}

// Any head size up to 256, any rotary_dim, any alignment: a warp a row, a lane every 32nd element.
template <typename T, bool PARTS>
__global__ void __launch_bounds__(THREADS) store_any_kernel(const Store s) {
  pdl_trigger();
  pdl_wait();
  constexpr int EACH = MOST_DIM / 32;
  const int heads = s.n_q + 2 * s.n_kv, lane = threadIdx.x & 31, half = s.rotary_dim / 2;
  const long long row = (long long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  if (row >= (long long)s.tokens * heads) return;
  const int token = (int)(row / heads), head = (int)(row - (long long)token * heads);
  const bool turns = head < s.n_q + s.n_kv, is_q = head < s.n_q;
  float x[EACH];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int i = j * 32 + lane;
    x[j] = 0.f;
    if (i >= s.d) continue;
    float own[1];
    take<T, PARTS, 1>(s, token, head * s.d + i, own);
    x[j] = own[0];
    if (turns && i < 2 * half) {
      const int pair = i < half ? i : i - half;
      float other[1];
      take<T, PARTS, 1>(s, token, head * s.d + (i < half ? i + half : i - half), other);
      const float2 f = s.table[(size_t)token * half + pair];
      if (is_q) {
        float rlo, rhi;
        rope_rotate(i < half ? own[0] : other[0], i < half ? other[0] : own[0], f.x, f.y, rlo, rhi);
        x[j] = i < half ? rlo : rhi;
      } else {
        const double a = own[0], b = other[0], c = f.x, n = f.y;
        x[j] = q8_to_odd(i < half ? a * c - b * n : a * c + b * n);
      }
    }
    top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
  }
  if (is_q) {
    T* to = static_cast<T*>(s.q_out) + (size_t)token * s.n_q * s.d + head * s.d;
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (j * 32 + lane < s.d) to[j * 32 + lane] = from_f32<T>(x[j]);
    return;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const bool is_v = !turns;
  const long long place = pool_row(s, token, head - s.n_q - (is_v ? s.n_kv : 0), lane == 0);
  if (place < 0) return;
  const int byte = q8_byte(top);
  const float inverse = byte == Q8_NAN_BYTE ? 0.f : q8_inverse(byte);
  uint8_t* to = (is_v ? s.v : s.k) + place * s.d;
#pragma unroll
  for (int j = 0; j < EACH; ++j)
    if (j * 32 + lane < s.d) to[j * 32 + lane] = (uint8_t)q8_encode2(byte == Q8_NAN_BYTE ? 0.f : x[j] * inverse, 0.f);
  if (lane == 0) (is_v ? s.v_scale : s.k_scale)[place] = (uint8_t)byte;
}

template <typename T, bool PARTS>
int launch_store(const Store& s, bool vec, cudaStream_t stream) {
  const long long rows = (long long)s.tokens * (s.n_q + 2 * s.n_kv);
  constexpr int N = PARTS ? 2 : 8, threads = PARTS ? FEW_THREADS : VEC_THREADS;
  if (vec) {
    const long long units = rows * (s.d / (2 * N));
    return (int)lab_launch(store_vec_kernel<T, PARTS, N>, dim3((unsigned)((units + threads - 1) / threads)), dim3(threads), 0, stream, s);
  }
  return (int)lab_launch(store_any_kernel<T, PARTS>, dim3((unsigned)((rows + THREADS / 32 - 1) / (THREADS / 32))), dim3(THREADS), 0, stream, s);
}

// ----------------------------------------------------------------------------------------
// Reading back: a thread takes N codes of a key and of a value and leaves 16 bytes of each (N = 1: any size and alignment).
// ----------------------------------------------------------------------------------------
// A thread keeps its place in the rows (so that what is divided is divided once) and takes EACH rows, their loads in flight together.
template <typename T, int N, int EACH>
__global__ void __launch_bounds__(THREADS) load_kernel(T* __restrict__ out_k, T* __restrict__ out_v, const uint8_t* __restrict__ k,
                                                       const uint8_t* __restrict__ v, const uint8_t* __restrict__ k_scale,
                                                       const uint8_t* __restrict__ v_scale, const int* __restrict__ slots, long long rows,
                                                       int n_kv, int d, int page_size, int num_pages) {
  pdl_trigger();
  pdl_wait();
  // a block: EACH passes of as many whole rows as it has threads for, or of a piece of a row
  const int pieces = d / N, width = n_kv * pieces, here = max(1, THREADS / width);
  const int sub = threadIdx.x / width, place = blockIdx.y * THREADS + (here > 1 ? threadIdx.x - sub * width : threadIdx.x);
  if (here > 1 ? sub >= here : place >= width) return;
  const int head = place / pieces, at = (place - head * pieces) * N;
  const long long row0 = (long long)blockIdx.x * here * EACH + (here > 1 ? sub : 0);
  const int shift = (page_size & (page_size - 1)) == 0 ? __ffs(page_size) - 1 : -1;
  long long from[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const long long row = row0 + i * here;
    const int slot = row < rows ? slots[row] : -1;
    const int page = slot < 0 ? -1 : shift >= 0 ? slot >> shift : slot / page_size;
    if (page >= num_pages && at == 0) lab_set_error(LAB_ERR_PAGE_RANGE);
    from[i] = page >= 0 && page < num_pages ? ((long long)page * n_kv + head) * page_size + (slot - page * page_size) : -1;
  }
  uint32_t kc[EACH][2], vc[EACH][2];
  float kf[EACH], vf[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    kc[i][0] = kc[i][1] = vc[i][0] = vc[i][1] = 0u;
    kf[i] = vf[i] = 0.f;
    if (from[i] < 0) continue;
    const uint8_t *kr = k + from[i] * d + at, *vr = v + from[i] * d + at;
    if constexpr (N == 8) {
      const uint2 x = *reinterpret_cast<const uint2*>(kr), y = *reinterpret_cast<const uint2*>(vr);
      kc[i][0] = x.x, kc[i][1] = x.y, vc[i][0] = y.x, vc[i][1] = y.y;
    } else if constexpr (N == 4) {
      kc[i][0] = *reinterpret_cast<const uint32_t*>(kr), vc[i][0] = *reinterpret_cast<const uint32_t*>(vr);
    } else {
      kc[i][0] = *kr, vc[i][0] = *vr;
    }
    kf[i] = q8_scale(k_scale[from[i]]), vf[i] = q8_scale(v_scale[from[i]]);
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const long long row = row0 + i * here;
    if (row >= rows) continue;
    const size_t to = ((size_t)row * n_kv + head) * d + at;
    auto one = [&](T* out, const uint32_t (&c)[2], float f) {
      const float4 x = q8_decode4(c[0]);
      if constexpr (N == 8) {
        const float4 y = q8_decode4(c[1]);
        const float z[8] = {x.x * f, x.y * f, x.z * f, x.w * f, y.x * f, y.y * f, y.z * f, y.w * f};
        put<8>(out + to, z);
      } else if constexpr (N == 4) {
        store4(out + to, make_float4(x.x * f, x.y * f, x.z * f, x.w * f));
      } else {
        out[to] = from_f32<T>(x.x * f);
      }
    };
    one(out_k, kc[i], kf[i]);
    one(out_v, vc[i], vf[i]);
  }
}

template <typename T>
int launch_load(T* out_k, T* out_v, const uint8_t* k, const uint8_t* v, const uint8_t* k_scale, const uint8_t* v_scale, const int* slots,
                long long rows, int n_kv, int d, int page_size, int num_pages, cudaStream_t stream) {
  constexpr int N = 16 / sizeof(T);
  const bool vec = d % N == 0 && ((((uintptr_t)out_k) | ((uintptr_t)out_v)) & 15) == 0 && ((((uintptr_t)k) | ((uintptr_t)v)) & (N - 1)) == 0;
  const long long width = (long long)n_kv * (vec ? d / N : d), here = width < THREADS ? THREADS / width : 1;
  const long long across = (width + THREADS - 1) / THREADS;
  // four rows a thread once every multiprocessor has two blocks of them (517 rows of 2 heads of 64, to bfloat16: 2.3 us by one
  // row a thread, 4.4 by four; 40,000 rows of 4 heads of 128, to 32 bits: 56 and 40)
  const bool four = rows / (here * 4) * across >= 2 * lab_sm_count();
  const long long blocks = (rows + here * (four ? 4 : 1) - 1) / (here * (four ? 4 : 1));
  if (blocks >= (1ll << 31) || across > 65535) return (int)cudaErrorInvalidValue;
  return (int)lab_launch(vec ? four ? load_kernel<T, N, 4> : load_kernel<T, N, 1> : four ? load_kernel<T, 1, 4> : load_kernel<T, 1, 1>,
                         dim3((unsigned)blocks, (unsigned)across), dim3(THREADS), 0, stream, out_k, out_v, k, v, k_scale, v_scale, slots, rows,
                         n_kv, d, page_size, num_pages);
}

}  // namespace

// A call, as the host packs it.  rows: [tokens, row_stride] of `dtype`, or (parts > 0) [parts, tokens, width] floats whose sum with
// `bias` is rounded to 32 bits and then to bfloat16 first; width = (n_q + 2 n_kv) d.  table: [tokens, rotary_dim / 2] (cos, sin).  q_out: [tokens, n_q *
// d].  Slots that are not negative differ from one another.
struct LabQ8Store {
  const void *rows, *bias, *table;
  const int* slots;
  void *q_out, *k, *v, *k_scale, *v_scale;
  long long row_stride, part_stride;
  int parts, rotary_dim, tokens, n_q, n_kv, d, page_size, num_pages, dtype;
};

LAB_EXPORT int lab_rope_kv_store_q8(const LabQ8Store* c, cudaStream_t stream) {
  if (c->tokens <= 0) return 0;
  const int parts = c->parts, d = c->d, rotary_dim = c->rotary_dim;
  if (d < 1 || d > MOST_DIM || rotary_dim < 0 || rotary_dim % 2 || rotary_dim > d || c->n_q < 0 || c->n_kv < 1 || c->page_size < 1 ||
      c->num_pages < 0 || (long long)c->tokens * (c->n_q + 2 * c->n_kv) * 32 >= (1ll << 31) || parts < 0 ||
      (parts > 0 && c->dtype != LAB_BF16) || (rotary_dim > 0 && c->table == nullptr))
    return (int)cudaErrorInvalidValue;
  Store s;
  s.rows = c->rows, s.row_stride = c->row_stride, s.parts = parts, s.part_stride = c->part_stride, s.bias = (const __nv_bfloat16*)c->bias;
  s.table = (const float2*)c->table, s.rotary_dim = rotary_dim, s.slots = c->slots, s.q_out = c->q_out;
  s.k = (uint8_t*)c->k, s.v = (uint8_t*)c->v, s.k_scale = (uint8_t*)c->k_scale, s.v_scale = (uint8_t*)c->v_scale;
  s.tokens = c->tokens, s.n_q = c->n_q, s.n_kv = c->n_kv, s.d = d, s.page_size = c->page_size, s.num_pages = c->num_pages;
  const int size = parts > 0 || c->dtype == LAB_F32 ? 4 : 2;
  const bool vec = rotary_dim == d && d >= 16 && d <= (parts > 0 ? 128 : 256) && (d & (d - 1)) == 0 && c->row_stride * size % 16 == 0 &&
                   (parts == 0 || c->part_stride * size % 16 == 0) &&
                   (((uintptr_t)c->rows | (uintptr_t)c->table | (uintptr_t)c->q_out | (uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0;
  if (c->dtype == LAB_F32) return launch_store<float, false>(s, vec, stream);
  return parts > 0 ? launch_store<__nv_bfloat16, true>(s, vec, stream) : launch_store<__nv_bfloat16, false>(s, vec, stream);
}

// out_k, out_v: [rows, n_kv, d] of `dtype`; a negative slot gives a row of zeros.
struct LabQ8Load {
  void *out_k, *out_v;
  const void *k, *v, *k_scale, *v_scale;
  const int* slots;
  long long rows;
  int n_kv, d, page_size, num_pages, dtype;
};

LAB_EXPORT int lab_kv_load_q8(const LabQ8Load* c, cudaStream_t stream) {
  if (c->rows <= 0) return 0;
  if (c->d < 1 || c->n_kv < 1 || c->page_size < 1 || c->num_pages < 0) return (int)cudaErrorInvalidValue;
  const uint8_t *k = (const uint8_t*)c->k, *v = (const uint8_t*)c->v, *ks = (const uint8_t*)c->k_scale, *vs = (const uint8_t*)c->v_scale;
  if (c->dtype == LAB_F32)
    return launch_load((float*)c->out_k, (float*)c->out_v, k, v, ks, vs, c->slots, c->rows, c->n_kv, c->d, c->page_size, c->num_pages, stream);
  return launch_load((__nv_bfloat16*)c->out_k, (__nv_bfloat16*)c->out_v, k, v, ks, vs, c->slots, c->rows, c->n_kv, c->d, c->page_size,
                     c->num_pages, stream);
}
