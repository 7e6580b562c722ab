// Drafted tokens against the target's probabilities.
//
// A request brings its rows of logits, one after the token it holds and one after each drafted token; draft x_i is judged by row
// i.  With p = softmax(logits / T) and q the probabilities that the draft was drawn from (or all of it on x_i):
//   accept x_i while u_i q(x_i) < p(x_i); at the first refusal, and after the last row, draw the token that ends the request:
//   argmax_t w_t / E_t with w = max(p - q, 0) at a refusal and w = p after the last row, E_t = -log(u_t) exponential.
// What comes out is distributed as the target's own draws are.  Where w is nothing anywhere (p = q up to rounding) w = p.
// T = 0: accept while x_i is the argmax of its row, and end with the argmax (ties: the smallest index; a NaN never wins, and a
// row without any number gives INT32_MAX, as the sampling kernel does).
// The u come from the sampling kernel's hash of (seed, position, t), so a draw depends on neither the batch nor the step; u_i of
// the test is the hash of the row's key's complement.  A draft that the sampler itself drew by the request's seed was chosen by the
// very E_t of its row: given that draft and its refusal they are no exponentials any more, and a draw by them favours what the draft
// passed over.  A call over such drafts says so (`fresh`), and the draw after a refusal then takes a key of its own, the hash of
// the row's.  (p = (.2, .5, .3), q = (.8, .05, .15), drafts of the sampler: (.2, .542, .258) by the row's key, p by one of its own.)
// The draw after the last row is the sampler's in either case.
//
// Probabilities are 32-bit.  p's relative error is about |logit / T| 2^-22 (the quotient's rounding, the largest logit's, and the
// fast exponential's 2^-22 of its argument) and 2^-20 for the rest; w = p - q keeps that error of p, so w's is p / w times as much.  A
// test or a draw goes another way than in exact arithmetic only where two numbers agree to that: to 2^-19 with logits of some ten
// and q away from p.
//
// Two launches: the rows' largest entry and sum of exponentials by chunk (every logit read once: the bound, memory), then a
// cluster of sixteen or four CTAs a request that puts its chunks together, each for itself, decides, and draws over the one row that
// is left (its logits come from L2).  Partial results lie in the caller's scratch and nothing has to be zero before a call, so calls
// on several streams, or from several graphs, do not meet.  (240 rows of 152,064, greedy: 24.7 us, 5.4 TB/s, 0.83 of a copy's rate;
// 8 requests of five rows, sampled: 17 us, the second launch the longer.)
#include <limits.h>

#include "common.cuh"

namespace {

constexpr int CHUNK = 8192, STAT_THREADS = 256, PICK_THREADS = 512, CLUSTER = 16, KEPT = 16;
constexpr int ROUNDS = CHUNK / (STAT_THREADS * 4);
constexpr uint32_t FRESH = 0x3C6EF372u;      // turns a row's key into that of the draw after its refusal (any pattern would do)

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7FEB352Du;
  x ^= x >> 15;
  x *= 0x846CA68Bu;
  x ^= x >> 16;
  return x;
}
__device__ __forceinline__ float uniform_of(uint32_t h) { return ((float)(h >> 9) + 0.5f) * (1.f / 8388608.f); }
__device__ __forceinline__ bool better(float v, int i, float bv, int bi) { return v > bv || (v == bv && i < bi); }

// Over a warp's lanes: the largest entry (none is NaN), the least index that has it, and the sum of exponentials relative to it.  The
// largest is found first, so that a lane forms one exponential and not two a step of the sum.  (The fast exponential: its error at
// x is about |x| 2^-22, and weighs e^x.)
__device__ __forceinline__ void warp_join(float& m, float& sum, int& at) {
  float big;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(big) : "f"(m));
  at = __reduce_min_sync(0xffffffffu, m == big ? at : INT_MAX);
  sum = warp_sum(m == big ? sum : sum * __expf(m - big));
  m = big;
}

struct Args {
  const float* logits;
  long long ld;
  const float* draft_probs;   // null: the drafts are certain
  long long ld_probs;
  const int *drafts, *starts;
  const float* temperature;   // [requests], null: all 0
  const uint32_t* seeds;
  const int* positions;       // of the token that a request's first row decides
  int rows, vocab, requests, chunks, fresh;
  float4* part;               // [rows, chunks]: largest entry, sum of exponentials relative to it, its index
  int *tokens, *counts;
};

// DRAWS false: every request is greedy.
template <bool DRAWS>
__global__ void __launch_bounds__(STAT_THREADS) verify_chunks_kernel(const Args a) {
  __shared__ float sm[STAT_THREADS / 32], ss[STAT_THREADS / 32];
  __shared__ int si[STAT_THREADS / 32];
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.y, chunk = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float* lr = a.logits + (size_t)row * a.ld;
  const int first = chunk * CHUNK, end = min(a.vocab, first + CHUNK);
  float x[4 * ROUNDS];
  const bool vec = (a.ld & 3) == 0 && (((uintptr_t)a.logits) & 15) == 0;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int i = first + (r * STAT_THREADS + (int)threadIdx.x) * 4;
    if (vec && i + 3 < end) {
      const float4 v = load4(lr + i);
      x[4 * r] = v.x, x[4 * r + 1] = v.y, x[4 * r + 2] = v.z, x[4 * r + 3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * r + e] = i + e < end ? lr[i + e] : __uint_as_float(0x7fffffffu);
    }
  }
  // the row's request, looked for while its entries arrive
  float inverse = 0.f;
  if constexpr (DRAWS) {
    int b = 0, past = a.requests;
    while (past - b > 1) {
      const int mid = (b + past) / 2;
      if (a.starts[mid] <= row) b = mid; else past = mid;
    }
    const float t = a.temperature[b];
    inverse = t > 0.f ? 1.f / t : 0.f;
  }
  const bool greedy = !DRAWS || inverse == 0.f;
  float m = -INFINITY;
  int at = INT_MAX;
  if (greedy) {
#pragma unroll
    for (int j = 0; j < 4 * ROUNDS; ++j) {
      const int i = first + ((j >> 2) * STAT_THREADS + (int)threadIdx.x) * 4 + (j & 3);
      if (better(x[j], i, m, at)) m = x[j], at = i;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4 * ROUNDS; ++j) {
      x[j] = fmaxf(x[j] * inverse, -INFINITY);      // (a NaN becomes -inf, the least of all)
      m = fmaxf(m, x[j]);
    }
  }
  float sum = 0.f;
  if (!greedy) {
    if (fabsf(m) < INFINITY) {
#pragma unroll
      for (int j = 0; j < 4 * ROUNDS; ++j) sum += __expf(x[j] - m);
    } else {      // all of them -inf, or some +inf: those that are the largest count
#pragma unroll
      for (int j = 0; j < 4 * ROUNDS; ++j) {
        const int i = first + ((j >> 2) * STAT_THREADS + (int)threadIdx.x) * 4 + (j & 3);
        sum += x[j] == m && i < end && lr[i] == lr[i] ? 1.f : 0.f;
      }
    }
  }
  warp_join(m, sum, at);
  if (lane == 0) sm[warp] = m, ss[warp] = sum, si[warp] = at;
  __syncthreads();
  if (warp != 0) return;
  constexpr int WARPS = STAT_THREADS / 32;
  const bool own = lane < WARPS;
  m = own ? sm[lane] : -INFINITY, sum = own ? ss[lane] : 0.f, at = own ? si[lane] : INT_MAX;
  warp_join(m, sum, at);
  if (lane != 0) return;
  a.part[(size_t)row * a.chunks + chunk] = make_float4(m, sum, __int_as_float(at), 0.f);
}

// A row's largest entry, its index, and its sum of exponentials, by one warp in the order of the chunks' lanes.
__device__ __forceinline__ float4 row_stats(const Args& a, int row, int lane) {
  float m = -INFINITY, sum = 0.f;
  int at = INT_MAX;
  for (int c = lane; c < a.chunks; c += 32) {
    const float4 p = a.part[(size_t)row * a.chunks + c];
    const int i = __float_as_int(p.z);
    const float big = fmaxf(m, p.x);
    sum = (m == big ? sum : sum * expf(m - big)) + (p.x == big ? p.y : p.y * expf(p.x - big));
    if (better(p.x, i, m, at)) at = i;
    m = big;
  }
  warp_join(m, sum, at);
  return make_float4(m, sum, __int_as_float(at), 0.f);
}

struct Best {
  float v, pv;      // of the weights left, and of p
  int i, pi;
  __device__ __forceinline__ void join(const Best& o) {
    if (better(o.v, o.i, v, i)) v = o.v, i = o.i;
    if (better(o.pv, o.pi, pv, pi)) pv = o.pv, pi = o.pi;
  }
};

// Two blocks a multiprocessor, up to 64 registers: sixteen at once are then found for each of eight requests.  (8 requests of four
// drafts, sampled: 16.9 us; 21.3 with 65 registers, where some cluster waits for another, 22.4 with blocks of 1,024.)
__global__ void __launch_bounds__(PICK_THREADS, 2) verify_pick_kernel(const Args a, int cluster) {
  __shared__ int stop_s;
  __shared__ float4 stats_s[KEPT + 1];      // the first rows' statistics, and those of the row that ends the request
  __shared__ Best warp_s[PICK_THREADS / 32];
  __shared__ Best cta_s[CLUSTER];
  pdl_trigger();
  if (cluster > 1) cluster_sync();      // every CTA is there before another writes to it
  pdl_wait();
  const int b = blockIdx.x / cluster, part = blockIdx.x - b * cluster, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // what a request has one of, asked for together
  const int lo = a.starts[b], hi = a.starts[b + 1];
  const float t = a.temperature != nullptr ? a.temperature[b] : 0.f;
  const uint32_t seed = a.temperature != nullptr ? a.seeds[b] : 0u;
  const int position = a.temperature != nullptr ? a.positions[b] : 0;
  const bool sound = lo >= 0 && hi <= a.rows && hi >= lo;      // rows ascending within the logits
  const int n = sound ? hi - lo : 0;
  const float inverse = t > 0.f ? 1.f / t : 0.f;
  const bool greedy = inverse == 0.f;
  if (threadIdx.x == 0) {
    stop_s = max(n - 1, 0);
    if (part == 0 && !sound) lab_set_error(LAB_ERR_ROW_RANGE);
  }
  __syncthreads();
  auto key_of = [&](int i) { return mix32(mix32(seed ^ 0x9E3779B9u) ^ (uint32_t)(position + i)); };
  for (int i = warp; i < n; i += PICK_THREADS / 32) {
    const int row = lo + i, x = a.drafts[row];
    const bool judged = i < n - 1, token = x >= 0 && x < a.vocab, gathers = judged && token && !greedy;
    const float logit = gathers ? a.logits[(size_t)row * a.ld + x] : 0.f;
    const float q = gathers && a.draft_probs != nullptr ? a.draft_probs[(size_t)row * a.ld_probs + x] : 1.f;
    const float4 s = row_stats(a, row, lane);
    bool taken = token;
    if (greedy) {
      taken = taken && x == __float_as_int(s.z);
    } else if (taken) {
      const float v = logit * inverse;
      const float p = (v == s.x ? 1.f : expf(v - s.x)) / s.y;
      taken = uniform_of(mix32(~key_of(i))) * q < p;
    }
    if (lane == 0) {
      if (judged && !taken) atomicMin(&stop_s, i);
      if (i < KEPT) stats_s[i] = s;
    }
  }
  __syncthreads();
  const int stop = stop_s, row = lo + stop;
  if (stop >= KEPT) {      // (a request of many drafts)
    if (warp == 0) {
      const float4 s = row_stats(a, row, lane);
      if (lane == 0) stats_s[KEPT] = s;
    }
    __syncthreads();
  }
  const float4 ends = stats_s[min(stop, KEPT)];
  Best best = {0.f, 0.f, INT_MAX, INT_MAX};      // a weight above 0 is wanted
  if (!greedy && n > 0) {
    const float m = ends.x, inverse_sum = 1.f / ends.y;
    const bool over = stop == n - 1;
    const uint32_t key = a.fresh && !over ? mix32(key_of(stop) ^ FRESH) : key_of(stop);
    const float* lr = a.logits + (size_t)row * a.ld;
    const float* qr = !over && a.draft_probs != nullptr ? a.draft_probs + (size_t)row * a.ld_probs : nullptr;
    const int certain = !over && a.draft_probs == nullptr ? a.drafts[row] : -1;
    // w / E <= w / (1 - u), so most entries are passed over without a logarithm: those that cannot beat what the warp has found.
    float least = 0.f, p_least = 0.f;
    auto consider = [&](float logit, float q, int i) {
      const float v = logit * inverse;
      const float p = (v == m ? 1.f : __expf(v - m)) * inverse_sum;
      const float w = i == certain ? 0.f : fmaxf(p - q, 0.f);
      const uint32_t h = mix32(key + (uint32_t)i * 0x85EBCA6Bu) >> 9;
      const float rest = (8388607.5f - (float)h) * (1.f / 8388608.f);      // 1 - u
      if (w >= least * rest || p >= p_least * rest) {
        const float rate = __fdividef(1.f, -logf(((float)h + 0.5f) * (1.f / 8388608.f)));
        if (better(w * rate, i, best.v, best.i)) best.v = w * rate, best.i = i;
        if (better(p * rate, i, best.pv, best.pi)) best.pv = p * rate, best.pi = i;
      }
    };
    const bool vec = (a.ld & 3) == 0 && (((uintptr_t)a.logits) & 15) == 0 &&
                     (qr == nullptr || ((a.ld_probs & 3) == 0 && (((uintptr_t)a.draft_probs) & 15) == 0));
    const int step = cluster * PICK_THREADS * 4;
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
    auto ask = [&](int i, float4& v, float4& q) {
      const bool whole = vec && i + 3 < a.vocab;
      v = whole ? load4(lr + i) : none;
      q = whole && qr != nullptr ? load4(qr + i) : none;
    };
    float4 v, q, v_next, q_next;
    ask(part * PICK_THREADS * 4 + (int)threadIdx.x * 4, v, q);
    for (int base = part * PICK_THREADS * 4; base < a.vocab; base += step) {
      const int i = base + (int)threadIdx.x * 4;
      ask(i + step, v_next, q_next);
      if (vec && i + 3 < a.vocab) {
        consider(v.x, q.x, i);
        consider(v.y, q.y, i + 1);
        consider(v.z, q.z, i + 2);
        consider(v.w, q.w, i + 3);
      } else {
        for (int e = i; e < min(i + 4, a.vocab); ++e) consider(lr[e], qr != nullptr ? qr[e] : 0.f, e);
      }
      v = v_next, q = q_next;
      // a little less than the best: what the bound's own rounding could lose
      least = warp_max(best.v) * 0.9999f;
      p_least = warp_max(best.pv) * 0.9999f;
    }
  }
  auto over_lanes = [&]() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Best other;
      other.v = __shfl_xor_sync(0xffffffffu, best.v, o), other.i = __shfl_xor_sync(0xffffffffu, best.i, o);
      other.pv = __shfl_xor_sync(0xffffffffu, best.pv, o), other.pi = __shfl_xor_sync(0xffffffffu, best.pi, o);
      best.join(other);
    }
  };
  over_lanes();
  if (lane == 0) warp_s[warp] = best;
  __syncthreads();
  if (warp == 0) {
    best = lane < PICK_THREADS / 32 ? warp_s[lane] : Best{0.f, 0.f, INT_MAX, INT_MAX};
    over_lanes();
    if (cluster > 1 && lane == 0) {
      const uint32_t to = map_to_rank(smem_u32(&cta_s[part]), 0);
      st_cluster_f32(to, best.v);
      st_cluster_f32(to + 4, best.pv);
      st_cluster_f32(to + 8, __int_as_float(best.i));
      st_cluster_f32(to + 12, __int_as_float(best.pi));
    }
  }
  if (cluster > 1) {
    cluster_sync();
    if (part != 0) return;
    if (warp == 0) {
      best = lane < cluster ? cta_s[lane] : Best{0.f, 0.f, INT_MAX, INT_MAX};
      over_lanes();
    }
  }
  if (n == 0) {
    if (threadIdx.x == 0) a.counts[b] = 0;
    return;
  }
  for (int i = threadIdx.x; i < n; i += PICK_THREADS)
    if (i != stop) a.tokens[lo + i] = i < stop ? a.drafts[lo + i] : -1;
  if (threadIdx.x == 0) {
    a.tokens[row] = greedy ? __float_as_int(ends.z) : best.v > 0.f ? best.i : best.pi;
    a.counts[b] = stop + 1;
  }
}

}  // namespace

// A call needs 16 bytes of scratch a row and chunk of this many entries.
LAB_EXPORT int lab_verify_chunk() { return CHUNK; }

// A call, as the host packs it.  logits [rows, vocab] 32-bit, rows `ld` apart; draft_probs likewise or null; drafts [rows]: the token
// drafted after a row's (a request's last row has none); starts [requests + 1]; temperature, seeds, positions [requests], null:
// greedy; fresh: the draw after a refusal takes random numbers of its own.  tokens [rows]: what a request's rows give, drafts that
// were accepted, the token that ends it, -1 behind it; counts [requests].
struct LabVerify {
  int *tokens, *counts;
  const float *logits, *draft_probs;
  const int *drafts, *starts;
  const float* temperature;
  const uint32_t* seeds;
  const int* positions;
  void* scratch;
  long long ld, ld_probs;
  int rows, vocab, requests, fresh;
};

LAB_EXPORT int lab_verify_drafts(const LabVerify* c, cudaStream_t stream) {
  const int rows = c->rows, vocab = c->vocab, requests = c->requests;
  void* scratch = c->scratch;
  const float* temperature = c->temperature;
  if (requests <= 0) return 0;
  if (rows < 0 || rows > 65535 || vocab < 1 || (rows > 0 && scratch == nullptr) || (((uintptr_t)scratch) & 15) ||
      (temperature != nullptr && (c->seeds == nullptr || c->positions == nullptr)))
    return (int)cudaErrorInvalidValue;
  Args a;
  a.logits = c->logits, a.ld = c->ld, a.draft_probs = c->draft_probs, a.ld_probs = c->ld_probs, a.drafts = c->drafts, a.starts = c->starts;
  a.temperature = temperature, a.seeds = c->seeds, a.positions = c->positions;
  a.rows = rows, a.vocab = vocab, a.requests = requests, a.fresh = c->fresh, a.chunks = (vocab + CHUNK - 1) / CHUNK;
  a.part = (float4*)scratch, a.tokens = c->tokens, a.counts = c->counts;
  if (rows > 0) {
    const cudaError_t e = lab_launch(temperature != nullptr ? verify_chunks_kernel<true> : verify_chunks_kernel<false>, dim3(a.chunks, rows), dim3(STAT_THREADS), 0, stream, a);
    if (e != cudaSuccess) return (int)e;
  }
  // Draws: sixteen CTAs a request while all of them find room, four beyond that, where each CTA's start is paid in turns (rows of
  // 151,936, five a request; 12 requests 19.2 us by sixteen and 23.6 by four, 18: 27.4 and 26.6, 48: 63 and 52, 128: 157 and 114;
  // by two 106 at 128, but 54 at 48).
  const int cluster = temperature == nullptr ? 1 : (long long)requests * CLUSTER <= 2 * lab_sm_count() ? CLUSTER : CLUSTER / 4;
  // a cluster beyond the portable size: asked for once per device
  static std::atomic<bool> allowed[LabShared::kDevices] = {};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return (int)e;
  if (device >= LabShared::kDevices || !allowed[device].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(verify_pick_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return (int)e;
    if (device < LabShared::kDevices) allowed[device].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(requests * cluster);
  cfg.blockDim = dim3(PICK_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_lab_pdl ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, verify_pick_kernel, a, cluster);
}
