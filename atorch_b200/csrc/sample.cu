// The next token of every row of logits: temperature, top-k, top-p and min-p, drawn with given waiting times.
//
// w = exp((x - max) / T). The tokens in the order (larger logit, lower index) that are left are a prefix of it: the first `top_k`; of
// these the ones whose predecessors weigh less than top_p of what they weigh together; of these the ones with w >= min_p. Drawn is the
// token with the largest w / waiting time.
#include "common.cuh"

namespace {
using namespace atb;

constexpr int THREADS = 512;

// Place in the order as a number: a greater one comes first. The logit, both zeros alike and a NaN as -inf, then the lower index.
ATB_DEVICE unsigned long long key_of(float x, unsigned index) {
  const uint32_t u = __float_as_uint((x != x ? -INFINITY : x) + 0.f);
  return ((unsigned long long)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32) | (0xffffffffu - index);
}
ATB_DEVICE double block_sum_d(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.;
  for (int i = 0; i < THREADS / 32; ++i) t += red[i];
  return t;
}

struct Args {
  const void* logits;
  const float* waiting;
  const float* t_rows;
  const int* k_rows;
  const float* p_rows;
  const float* m_rows;
  long long* tokens;
  float* logprobs;
  int V;
  long long stride, wait_stride;
  double t, p, m;
  int k;
  const int* status;
};

// One block a row, everything in 64 bits. The end of the prefix is found bit by bit: is what reaches a key still too much?
template <typename T>
__global__ void __launch_bounds__(THREADS) sample_kernel(Args a) {
  __shared__ double red[THREADS / 32];
  __shared__ double best_score[THREADS];
  __shared__ int best_at[THREADS];
  grid_go();
  grid_wait();
  const long long row = blockIdx.x;
  const T* const x = (const T*)a.logits + row * a.stride;
  const float* const wait = a.waiting + row * a.wait_stride;
  double temp = a.t_rows ? a.t_rows[row] : a.t, p = a.p_rows ? a.p_rows[row] : a.p, m = a.m_rows ? a.m_rows[row] : a.m;
  int k = a.k_rows ? a.k_rows[row] : a.k;
  const int V = a.V;
  unsigned long long first = 0;
  for (int i = threadIdx.x; i < V; i += THREADS) first = max(first, key_of(to_f32<T>(x[i]), i));
  __shared__ unsigned long long keys[THREADS];
  keys[threadIdx.x] = first;
  __syncthreads();
  for (int i = 0; i < THREADS; ++i) first = max(first, keys[i]);
  const int first_at = (int)(0xffffffffu - (uint32_t)first);
  const float top = to_f32<T>(x[first_at]);
  if (*a.status != 0 || !(top > -INFINITY) || !(temp > 0.)) {
    if (threadIdx.x == 0) {
      a.tokens[row] = top > -INFINITY && *a.status == 0 ? first_at : 0;
      a.logprobs[row] = top > -INFINITY && *a.status == 0 ? 0.f : -INFINITY;
    }
    return;
  }
  auto weight = [&](float v) { return v == top ? 1. : v > -INFINITY ? exp(((double)v - (double)top) / temp) : 0.; };
  unsigned long long last = 0;        // keys of at least this are left
  // the greatest key such that `enough` of what reaches it
  auto cut = [&](auto enough) {
    unsigned long long c = 0;
    for (int bit = 63; bit >= 0; --bit)
      if (enough(c | 1ull << bit)) c |= 1ull << bit;
    return c;
  };
  if (k > 0 && k < V)
    last = cut([&](unsigned long long c) {
      double n = 0.;
      for (int i = threadIdx.x; i < V; i += THREADS) n += key_of(to_f32<T>(x[i]), i) >= c;
      return block_sum_d(n, red) >= k;
    });
  auto sum_from = [&](unsigned long long c) {
    double n = 0.;
    for (int i = threadIdx.x; i < V; i += THREADS)
      if (key_of(to_f32<T>(x[i]), i) >= c) n += weight(to_f32<T>(x[i]));
    return block_sum_d(n, red);
  };
  if (p < 1.) {
    const double share = p * sum_from(last);
    const unsigned long long c = cut([&](unsigned long long c) { return sum_from(c) >= share && c <= first; });
    last = max(last, c);
  }
  double sum = 0., score = -1.;
  int at = V;
  for (int i = threadIdx.x; i < V; i += THREADS) {
    const double w = weight(to_f32<T>(x[i]));
    if (key_of(to_f32<T>(x[i]), i) < last || w < m || w == 0.) continue;
    const float t = wait[i];
    const double s = t >= 0.f ? w / (double)t : 0.;
    sum += w;
    if (s > score) {
      score = s;
      at = i;
    }
  }
  sum = block_sum_d(sum, red);
  best_score[threadIdx.x] = score;
  best_at[threadIdx.x] = at;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < THREADS; ++i)
      if (best_score[i] > score || (best_score[i] == score && best_at[i] < at)) {
        score = best_score[i];
        at = best_at[i];
      }
    a.tokens[row] = at;
    a.logprobs[row] = (float)log(weight(to_f32<T>(x[at])) / sum);
  }
}
}  // namespace

// t, p, m: the bits of fp64 numbers
extern "C" int atb_sample(const void* logits, const void* waiting, const void* t_rows, const void* k_rows, const void* p_rows,
                          const void* m_rows, void* tokens, void* logprobs, int rows, int V, long long stride, long long wait_stride,
                          long long t, long long p, long long m, int k, int dtype, void* stream, void* status) {
  if (rows <= 0) return 0;
  auto number = [](long long bits) {
    double d;
    __builtin_memcpy(&d, &bits, 8);
    return d;
  };
  const Args a{logits, (const float*)waiting, (const float*)t_rows, (const int*)k_rows, (const float*)p_rows, (const float*)m_rows,
               (long long*)tokens, (float*)logprobs, V, stride, wait_stride, number(t), number(p), number(m), k, (const int*)status};
  const cudaStream_t st = (cudaStream_t)stream;
  if (dtype == 0) return launched(launch_after(sample_kernel<__nv_bfloat16>, dim3(rows), THREADS, 0, st, 1, a));
  if (dtype == 1) return launched(launch_after(sample_kernel<__half>, dim3(rows), THREADS, 0, st, 1, a));
  if (dtype == 2) return launched(launch_after(sample_kernel<float>, dim3(rows), THREADS, 0, st, 1, a));
  return -1;
}
