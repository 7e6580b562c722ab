// Attention over the paged 8-bit cache (quant8.cuh) on the ordinary units: any head size up to 256, any page size, queries of
// either storage type (32-bit queries: 32-bit arithmetic throughout).  What the tensor-core kernels do not take runs here.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - max_j),   j visible: first(pos_i) <= j <= min(pos_i, len - 1)
//
// A block takes one row and query head.  Its four warps take 32 keys in turn: a lane forms the score of its key (the codes of a
// key are read where they lie; the lanes' rows are neighbours in a page, so a line serves several of their reads), then the warp
// adds the 32 values, a lane every 32nd entry.  Running maximum, sum and accumulator are 32-bit, merged over the warps at the
// end.  Keys that a row does not see are not read.  Bound by instructions, about
// seven a byte: it is the fallback, and the tests' second opinion.
#include "quant8.cuh"

namespace {

constexpr int WARPS = 4, MOST_DIM = 256;

template <typename T>
__global__ void __launch_bounds__(32 * WARPS) attention_q8_any_kernel(
    T* __restrict__ out, long long out_stride, const T* __restrict__ q, long long q_stride, const uint8_t* __restrict__ k,
    const uint8_t* __restrict__ v, const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
    const int* __restrict__ q_start, const int* __restrict__ kv_len, const int* __restrict__ pos0, const int* __restrict__ block_table,
    int max_blocks, int requests, int n_q, int n_kv, int d, int page_size, int num_pages, int window, float scale) {
  constexpr int EACH = MOST_DIM / 32;
  __shared__ float qs[MOST_DIM], acc_s[WARPS][MOST_DIM], max_s[WARPS], sum_s[WARPS];
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the request whose rows hold row t: the last that starts at or before it (requests without rows share a start)
  int b = 0, past = requests;
  while (past - b > 1) {
    const int mid = (b + past) / 2;
    if (q_start[mid] <= t) b = mid; else past = mid;
  }
  if (t < q_start[b] || t >= q_start[b + 1]) return;      // a row of no request stays as it is
  const int pos = pos0[b] + t - q_start[b], last = min(pos, kv_len[b] - 1), first = lab_first_key(pos, window);
  const int* bt = block_table + (size_t)b * max_blocks;
  const int kvh = h / (n_q / n_kv);
  for (int i = threadIdx.x; i < d; i += 32 * WARPS) qs[i] = to_f32(q[(size_t)t * q_stride + (size_t)h * d + i]) * scale;
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) acc[e] = 0.f;
  for (int base = first / 32 * 32 + warp * 32; base <= last; base += 32 * WARPS) {
    const int j = base + lane;
    long long row = -1;
    if (j >= first && j <= last && j / page_size < max_blocks) {
      const int page = bt[j / page_size];
      if (page < 0 || page >= num_pages) lab_set_error(LAB_ERR_PAGE_RANGE);      // a page that holds visible keys must exist
      else row = ((long long)page * n_kv + kvh) * page_size + j % page_size;
    }
    float s = -INFINITY;
    if (row >= 0) {
      const uint8_t* kr = k + row * d;
      float dot = 0.f;
      if (d % 16 == 0 && (((uintptr_t)k) & 15) == 0) {
        for (int i = 0; i < d; i += 16) {
          const uint4 c = *reinterpret_cast<const uint4*>(kr + i);
          const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 x = q8_decode4(w[e]);
            dot = fmaf(x.x, qs[i + 4 * e], fmaf(x.y, qs[i + 4 * e + 1], fmaf(x.z, qs[i + 4 * e + 2], fmaf(x.w, qs[i + 4 * e + 3], dot))));
          }
        }
      } else {
        for (int i = 0; i < d; ++i) dot = fmaf(q8_decode(kr[i]), qs[i], dot);
      }
      s = dot * q8_scale(k_scale[row]);
    }
    // fmaxf passes over a NaN: the maximum stays a number, and the NaN reaches the sums through its own p
    const float m_new = fmaxf(m, warp_max(s)), held = m_new == -INFINITY ? 0.f : m_new;
    const float f = m == -INFINITY ? 0.f : expf(m - held);
    const float p = row >= 0 ? expf(s - held) : 0.f;
    const float w = row >= 0 ? p * q8_scale(v_scale[row]) : 0.f;
    l = l * f + warp_sum(p);
    m = m_new;
#pragma unroll
    for (int e = 0; e < EACH; ++e) acc[e] *= f;
    for (int i = 0; i < 32; ++i) {
      const long long ri = __shfl_sync(0xffffffffu, row, i);
      const float wi = __shfl_sync(0xffffffffu, w, i);
      if (ri < 0) continue;
#pragma unroll
      for (int e = 0; e < EACH; ++e)
        if (e * 32 + lane < d) acc[e] = fmaf(wi, q8_decode(v[ri * d + e * 32 + lane]), acc[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (e * 32 + lane < d) acc_s[warp][e * 32 + lane] = acc[e];
  if (lane == 0) max_s[warp] = m, sum_s[warp] = l;
  __syncthreads();
  float big = -INFINITY;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) big = fmaxf(big, max_s[w]);
  float den = 0.f, share[WARPS];
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    share[w] = max_s[w] == -INFINITY ? 0.f : expf(max_s[w] - big);
    den += max_s[w] == -INFINITY ? sum_s[w] : share[w] * sum_s[w];      // (no number above -inf: 0, or NaN from NaN scores alone)
  }
  for (int i = threadIdx.x; i < d; i += 32 * WARPS) {
    float num = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) num = fmaf(share[w], acc_s[w][i], num);
    out[(size_t)t * out_stride + (size_t)h * d + i] = from_f32<T>(den == 0.f ? 0.f : num / den);
  }
}

}  // namespace

// A call, as the host packs it.  q: `tokens` rows q_stride elements apart, out likewise, both of `dtype`.  window as lab_first_key
// takes it.
struct LabQ8Any {
  void* out;
  const void *q, *k, *v, *k_scale, *v_scale;
  const int *q_start, *kv_len, *pos0, *block_table;
  long long out_stride, q_stride;
  int tokens, max_blocks, requests, n_q, n_kv, d, page_size, num_pages, window, dtype;
  float scale;
};

LAB_EXPORT int lab_attention_q8_any(const LabQ8Any* c, cudaStream_t stream) {
  if (c->tokens <= 0 || c->requests <= 0) return 0;
  if (c->d < 1 || c->d > MOST_DIM || c->n_kv < 1 || c->n_q < 1 || c->n_q % c->n_kv || c->n_q > 65535 || c->page_size < 1 || c->num_pages < 0 ||
      c->max_blocks < 0)
    return (int)cudaErrorInvalidValue;
  auto launch = [&](auto kernel, auto* o, auto* x) {
    return (int)lab_launch(kernel, dim3(c->tokens, c->n_q), dim3(32 * WARPS), 0, stream, o, c->out_stride, x, c->q_stride, (const uint8_t*)c->k,
                           (const uint8_t*)c->v, (const uint8_t*)c->k_scale, (const uint8_t*)c->v_scale, c->q_start, c->kv_len, c->pos0,
                           c->block_table, c->max_blocks, c->requests, c->n_q, c->n_kv, c->d, c->page_size, c->num_pages, c->window, c->scale);
  };
  if (c->dtype == LAB_F32) return launch(attention_q8_any_kernel<float>, (float*)c->out, (const float*)c->q);
  return launch(attention_q8_any_kernel<__nv_bfloat16>, (__nv_bfloat16*)c->out, (const __nv_bfloat16*)c->q);
}
