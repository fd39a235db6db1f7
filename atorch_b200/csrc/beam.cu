// One step of a beam search: the best continuations over beams and vocabulary, and the paged cache's move to its new beams.
//
// A continuation of beam w by token v has f = score[w] + (x[w, v] - lse(x[w])), evaluated in fp32 in this order; NaN counts as
// -inf. The `keep` largest f of a sequence's beams are kept, equal ones by the lower w, then the lower v.
#include "common.cuh"

namespace {
using namespace atb;

constexpr int THREADS = 512, MOST = 32, ROOM = 1024;      // threads of a row, beams, candidates that a row has room for

// A number whose order as an unsigned integer is that of f (both zeros alike), then of the lower index.
ATB_DEVICE unsigned long long key_of(float f, unsigned index) {
  uint32_t u = __float_as_uint(f + 0.f);
  u = u & 0x80000000u ? ~u : u | 0x80000000u;
  return ((unsigned long long)u << 32) | (0xffffffffu - index);
}
ATB_DEVICE float value_of(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
ATB_DEVICE unsigned index_of(unsigned long long key) { return 0xffffffffu - (uint32_t)key; }

ATB_DEVICE float total(float score, float x, float lse) {
  const float f = __fadd_rn(score, __fsub_rn(x, lse));
  return f != f ? -INFINITY : f;
}

ATB_DEVICE unsigned long long block_max_key(unsigned long long k, unsigned long long* red) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(0xffffffffu, k, o);
    k = x > k ? x : k;
  }
  __syncthreads();
  if (lane == 0) red[w] = k;
  __syncthreads();
  unsigned long long t = lane < (int)(blockDim.x >> 5) ? red[lane] : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(0xffffffffu, t, o);
    t = x > t ? x : t;
  }
  return t;
}

// Calls f(value, index) for the elements of a row that this thread has: 16-byte pieces where the row allows it.
template <typename T, typename F>
ATB_DEVICE void each(const T* row, int V, bool wide, F f) {
  constexpr int N = 16 / sizeof(T);
  const int pieces = wide ? V / N : 0;
  for (int i = threadIdx.x; i < pieces; i += THREADS) {
    const uint4 u = reinterpret_cast<const uint4*>(row)[i];
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int e = 0; e < N; ++e) f(to_f32<T>(h[e]), i * N + e);
  }
  for (int i = pieces * N + threadIdx.x; i < V; i += THREADS) f(to_f32<T>(row[i]), i);
}

// The `keep` best continuations of one beam (a block), best first, as keys of f and token.
template <typename T>
__global__ void __launch_bounds__(THREADS) beam_row_kernel(const T* logits, const float* scores, const unsigned char* finished,
                                                           unsigned long long* best, int V, long long row_stride, int wide,
                                                           int eos, int keep, const int* status) {
  __shared__ float red[33];
  __shared__ unsigned long long red_key[THREADS / 32], room[ROOM], tops[THREADS];
  __shared__ int count;
  grid_go();
  grid_wait();
  if (__syncthreads_or(threadIdx.x == 0 && *status != 0)) return;
  const long long row = blockIdx.x;
  const float score = scores[row];
  unsigned long long* out = best + row * keep;
  const int n = min(keep, V);                      // what the row has; the rest is below everything
  for (int i = n + threadIdx.x; i < keep; i += THREADS) out[i] = 0;
  if (finished && finished[row]) {
    // only the end token goes on, at no cost; the others are impossible, and stand in their order
    for (int i = threadIdx.x; i < n; i += THREADS) {
      if (score == -INFINITY || score != score) out[i] = key_of(-INFINITY, i);
      else out[i] = i == 0 ? key_of(score, eos) : key_of(-INFINITY, i - 1 < eos ? i - 1 : i);
    }
    return;
  }
  if (score == -INFINITY || score != score) {
    for (int i = threadIdx.x; i < n; i += THREADS) out[i] = key_of(-INFINITY, i);
    return;
  }
  const T* x = logits + row * row_stride;
  float top = -INFINITY;
  bool bad = false;
  each<T>(x, V, wide, [&](float v, int) {
    top = fmaxf(top, v);
    bad = bad || v != v;
  });
  const float row_top = block_max(top, red);
  float sum = 0.f;
  each<T>(x, V, wide, [&](float v, int) { sum += expf(v - row_top); });
  sum = block_sum(sum, red);
  float lse = row_top + logf(sum);
  if (__syncthreads_or(bad)) lse = __int_as_float(0x7fc00000);      // a NaN makes every f of the row one

  // the n-th largest of the threads' maxima: no fewer than n continuations reach it
  tops[threadIdx.x] = key_of(total(score, top, lse), threadIdx.x);
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  int rank = 0;
  for (int i = 0; i < THREADS; ++i) rank += tops[i] > tops[threadIdx.x];
  if (rank == n - 1) red[32] = value_of(tops[threadIdx.x]);
  __syncthreads();
  const float least = red[32];
  if (least > -INFINITY) {
    each<T>(x, V, wide, [&](float v, int i) {
      const float f = total(score, v, lse);
      if (f >= least) {
        const int at = atomicAdd(&count, 1);
        if (at < ROOM) room[at] = key_of(f, i);
      }
    });
  } else if (threadIdx.x == 0) {
    count = ROOM + 1;
  }
  __syncthreads();
  const int have = count;
  if (have <= ROOM) {
    for (int i = threadIdx.x; i < have; i += THREADS) {
      const unsigned long long k = room[i];
      int place = 0;
      for (int j = 0; j < have; ++j) place += room[j] > k;
      if (place < n) out[place] = k;
    }
    return;
  }
  // too many reach it, or too few continuations are possible at all: one after another
  unsigned long long last = ~0ull;
  for (int k = 0; k < n; ++k) {
    unsigned long long mine = 0;
    each<T>(x, V, wide, [&](float v, int i) {
      const unsigned long long key = key_of(total(score, v, lse), i);
      if (key < last && key > mine) mine = key;
    });
    last = block_max_key(mine, red_key);
    if (threadIdx.x == 0) out[k] = last;
  }
}

// The best of a sequence's beams (a block): each of the W keep continuations counts those before it.
__global__ void __launch_bounds__(256) beam_join_kernel(const unsigned long long* best, const unsigned char* finished,
                                                        float* scores, long long* tokens, int* parents,
                                                        unsigned char* ended, int W, int keep, int eos, const int* status) {
  __shared__ unsigned long long all[MOST * MOST];
  grid_go();
  grid_wait();
  if (__syncthreads_or(threadIdx.x == 0 && *status != 0)) return;
  const long long b = blockIdx.x;
  const int n = W * keep;
  for (int i = threadIdx.x; i < n; i += 256) all[i] = best[b * n + i];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 256) {
    const unsigned long long k = all[i];
    const int w = i / keep;
    int place = 0;
    for (int j = 0; j < n && place < keep; ++j) {
      // by f, then beam, then token (the low half of a key); within a beam the list is in order
      const unsigned long long o = all[j];
      const uint32_t fo = (uint32_t)(o >> 32), fk = (uint32_t)(k >> 32);
      place += fo != fk ? fo > fk : j < i;
    }
    if (place >= keep || k == 0) continue;
    const long long at = b * keep + place;
    scores[at] = value_of(k);
    tokens[at] = index_of(k);
    parents[at] = w;
    ended[at] = (finished && finished[b * W + w]) || (int)index_of(k) == eos;
  }
}

// The cache follows its beams: row b W + w of the table takes the full pages of row b W + parent[w], and its own last page the
// tokens of that row's last page. A thread has one place of all W rows and reads them all before it writes any, so the rows may
// change places. Bound by memory: each token of the last pages that moves is read and written once.
template <int MAX_W>
__global__ void __launch_bounds__(256) beam_reorder_kernel(uint8_t* codes, uint8_t* scales, int* table, const int* lengths,
                                                           const int* parents, int W, int width, long long table_stride,
                                                           int pages, long long page_bytes, long long scale_bytes,
                                                           int kv_heads, int page_shift, int token_bytes, int* status) {
  grid_go();
  grid_wait();
  if (__syncthreads_or(threadIdx.x == 0 && *status != 0)) return;
  const long long b = blockIdx.y, first = b * W;
  const int layer = (int)blockIdx.z - 1, n = lengths[first], full = n >> page_shift, rest = n - (full << page_shift);
  int from[MAX_W];
  bool good = n >= 0 && full + (rest > 0) <= width;
#pragma unroll
  for (int w = 0; w < MAX_W; ++w) {
    from[w] = w < W ? parents[first + w] : w;
    good = good && (w >= W || (from[w] >= 0 && from[w] < W && lengths[first + w] == n));
  }
  if (!good) {
    if (threadIdx.x == 0) atomicCAS(status, 0, (int)ATB_ERR_BAD_INDEX);
    return;
  }
  if (layer < 0) {                // the table
    for (int i = blockIdx.x * 256 + threadIdx.x; i < full; i += gridDim.x * 256) {
      int x[MAX_W];
#pragma unroll
      for (int w = 0; w < MAX_W; ++w)
        if (w < W) x[w] = table[(first + from[w]) * table_stride + i];
#pragma unroll
      for (int w = 0; w < MAX_W; ++w)
        if (w < W && from[w] != w) table[(first + w) * table_stride + i] = x[w];
    }
    return;
  }
  if (rest == 0) return;
  int page[MAX_W];
#pragma unroll
  for (int w = 0; w < MAX_W; ++w) {
    page[w] = w < W ? table[(first + w) * table_stride + full] : 0;
    good = good && page[w] >= 0 && page[w] < pages;
  }
  if (!good) {
    if (threadIdx.x == 0) atomicCAS(status, 0, (int)ATB_ERR_BAD_INDEX);
    return;
  }
  int source[MAX_W];              // page of the parent
#pragma unroll
  for (int w = 0; w < MAX_W; ++w) {
    source[w] = 0;
#pragma unroll
    for (int o = 0; o < MAX_W; ++o) source[w] = from[w] == o ? page[o] : source[w];
  }
  const int per_token = token_bytes / 16, per_head = rest * per_token, code_pieces = 2 * kv_heads * per_head;
  const int head_bytes = token_bytes << page_shift, all = code_pieces + kv_heads * rest;
  uint8_t* const layer_codes = codes + (long long)layer * pages * page_bytes;
  uint8_t* const layer_scales = scales + (long long)layer * pages * scale_bytes;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < all; i += gridDim.x * 256) {
    if (i < code_pieces) {
      const int h = i / per_head;
      const long long at = (long long)h * head_bytes + (i - h * per_head) * 16;
      uint4 x[MAX_W];
#pragma unroll
      for (int w = 0; w < MAX_W; ++w)
        if (w < W && from[w] != w) x[w] = *reinterpret_cast<const uint4*>(layer_codes + source[w] * page_bytes + at);
#pragma unroll
      for (int w = 0; w < MAX_W; ++w)
        if (w < W && from[w] != w) *reinterpret_cast<uint4*>(layer_codes + page[w] * page_bytes + at) = x[w];
    } else {
      const int j = i - code_pieces, h = j / rest;
      const long long at = ((long long)h << (page_shift + 3)) + (j - h * rest) * 8;
      uint2 x[MAX_W];
#pragma unroll
      for (int w = 0; w < MAX_W; ++w)
        if (w < W && from[w] != w) x[w] = *reinterpret_cast<const uint2*>(layer_scales + source[w] * scale_bytes + at);
#pragma unroll
      for (int w = 0; w < MAX_W; ++w)
        if (w < W && from[w] != w) *reinterpret_cast<uint2*>(layer_scales + page[w] * scale_bytes + at) = x[w];
    }
  }
}
}  // namespace

extern "C" int atb_beam_select(const void* logits, const void* scores, const void* finished, void* best, void* out_scores,
                               void* tokens, void* parents, void* ended, int B, int W, int V, long long row_stride, int wide,
                               int eos, int keep, int dtype, void* stream, void* status) {
  if (B <= 0 || keep <= 0) return 0;
  if (W < 1 || W > MOST || keep > MOST || V < 1 || (long long)B * W > 0x7fffffffLL) return -1;
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t rc = cudaErrorInvalidValue;
#define ROWS(T)                                                                                                          \
  rc = launch_after(beam_row_kernel<T>, dim3(B * W), THREADS, 0, st, 1, (const T*)logits, (const float*)scores,           \
                    (const unsigned char*)finished, (unsigned long long*)best, V, row_stride, wide, eos, keep, (const int*)status)
  if (dtype == 0) ROWS(__nv_bfloat16);
  if (dtype == 1) ROWS(__half);
  if (dtype == 2) ROWS(float);
#undef ROWS
  if (rc != cudaSuccess) return -5;
  return launch_after(beam_join_kernel, dim3(B), 256, 0, st, 1, (const unsigned long long*)best, (const unsigned char*)finished,
                      (float*)out_scores, (long long*)tokens, (int*)parents, (unsigned char*)ended, W, keep, eos,
                      (const int*)status) == cudaSuccess ? 0 : -5;
}

extern "C" int atb_beam_reorder(void* codes, void* scales, void* table, const void* lengths, const void* parents, int B, int W,
                                int width, long long table_stride, int layers, int pages, int kv_heads, int page_shift,
                                int head_dim, void* stream, void* status) {
  if (B <= 0 || W <= 0) return 0;
  if (W > MOST || B > 65535 || layers > 65534 || head_dim % 32) return -1;
  const int token_bytes = head_dim / 2;
  const long long page_bytes = (2LL * kv_heads * token_bytes) << page_shift, scale_bytes = (8LL * kv_heads) << page_shift;
  const long long most = (2LL * kv_heads * token_bytes / 16 + kv_heads) << page_shift;
  if (page_bytes > 0x7fffffffLL || most > 0x7fffffffLL) return -2;
  const dim3 grid((unsigned)((most + 255) / 256), B, layers + 1);
  cudaError_t rc;
#define MOVE(MAX_W)                                                                                                        \
  rc = launch_after(beam_reorder_kernel<MAX_W>, grid, 256, 0, (cudaStream_t)stream, 1, (uint8_t*)codes, (uint8_t*)scales,    \
                    (int*)table, (const int*)lengths, (const int*)parents, W, width, table_stride, pages, page_bytes,       \
                    scale_bytes, kv_heads, page_shift, token_bytes, (int*)status)
  if (W <= 4) MOVE(4);
  else if (W <= 8) MOVE(8);
  else if (W <= 16) MOVE(16);
  else MOVE(32);
#undef MOVE
  return rc == cudaSuccess ? 0 : -5;
}
