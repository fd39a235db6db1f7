// Paged key/value cache in 16 bits: append with rotation, attention of the newest tokens, eviction of tokens with little weight.
//
// One layer's cache is T [pages][2][kv heads][page size][D]: 0: keys, 1: values.
#include "paged.cuh"

namespace {
using namespace atb;

struct Cache : Paging {
  void* data;
};
template <typename T, int D>
ATB_DEVICE T* row_at(const Cache& c, int page, int which, int head, int slot) {
  return (T*)c.data + (((((long long)page * 2 + which) * c.kv_heads + head) << c.page_shift) + slot) * D;
}

// ----------------------------------------------------------------------------------
// Append
// ----------------------------------------------------------------------------------
constexpr int SMALL = 128;      // threads of a block: a few heads of one token

// A head of a token is D / 16 lanes: each has 8 dims of the first half and the 8 of the second half that they turn with. The
// rotation is that of separately rounded fp32 operations (no fused multiply-add), so that it does not depend on how a compiler
// contracts it. Bound by memory where there are many tokens, by latency for the one token of a step.
template <typename T, int D, int PER>
__global__ void __launch_bounds__(SMALL) kv_append_kernel(const T* qkv, T* q_out, T* k_out, Cache c, const int* seq, const int* pos,
                                                          const int* angles, const float* cosT, const float* sinT, int positions,
                                                          int n_q, long long token_stride, int* status) {
  grid_go();
  grid_wait();
  constexpr int L = D / 16, HALF = D / 2, EACH = SMALL / L;
  const int heads = n_q + 2 * c.kv_heads, l = threadIdx.x % L, h0 = blockIdx.y * (EACH * PER) + threadIdx.x / L;
  const long long t = blockIdx.x;
  const int before = *status, row = seq ? seq[t] : (int)t;
  int p = pos[t], page = -1;
  const int angle = angles ? angles[t] : p;
  uint4 x[PER][2];                 // 8 dims of the first half of head h0 + j EACH, 8 of the second
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (h0 + j * EACH < heads) {
      const T* src = qkv + t * token_stride + (long long)(h0 + j * EACH) * D + l * 8;
      x[j][0] = *reinterpret_cast<const uint4*>(src);
      x[j][1] = *reinterpret_cast<const uint4*>(src + HALF);
    }
  if (p >= 0) {
    page = page_of(c, row, p);
    if (page < 0 || (cosT && (angle < 0 || angle >= positions))) {
      atomicCAS(status, 0, (int)ATB_ERR_BAD_INDEX);
      page = -1;
      p = -1;
    }
  }
  float cs[8], sn[8];
  const bool turn = cosT && p >= 0 && h0 < n_q + c.kv_heads;
  if (turn) {
    load8<float>(cosT + (long long)angle * HALF + l * 8, cs);
    load8<float>(sinT + (long long)angle * HALF + l * 8, sn);
  }
  if (before != 0) return;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int h = h0 + j * EACH;
    if (h >= heads) break;
    if (turn && h < n_q + c.kv_heads) {
      T* const u = reinterpret_cast<T*>(&x[j][0]);
      T* const v = reinterpret_cast<T*>(&x[j][1]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = to_f32<T>(u[i]), b = to_f32<T>(v[i]);
        u[i] = from_f32<T>(__fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(b, sn[i])));
        v[i] = from_f32<T>(__fadd_rn(__fmul_rn(b, cs[i]), __fmul_rn(a, sn[i])));
      }
    }
    const int which = h >= n_q + c.kv_heads, head = h - n_q - (which ? c.kv_heads : 0);
    auto store = [&](T* dst) {
      *reinterpret_cast<uint4*>(dst + l * 8) = x[j][0];
      *reinterpret_cast<uint4*>(dst + HALF + l * 8) = x[j][1];
    };
    if (h < n_q) store(q_out + (t * n_q + h) * D);
    else if (!which && k_out) store(k_out + (t * c.kv_heads + head) * D);
    if (h >= n_q && page >= 0) store(row_at<T, D>(c, page, which, head, p & ((1 << c.page_shift) - 1)));
  }
}

// ----------------------------------------------------------------------------------
// Attention
// ----------------------------------------------------------------------------------
struct AttnArgs {
  Cache c;
  const int* lengths;
  const void* q;
  void* out;
  float* lse;                 // [rows][heads][S] or nullptr
  float* weights;             // [rows][kv heads][places] or nullptr
  float* partial;
  long long places, q_batch, q_token;
  int S, heads, group;
  float scale_log2;           // softmax scale * log2(e)
  int* status;
};

// One query of one head: a block's warps take its keys in turn, a lane D / 32 dims.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv_attention_kernel(AttnArgs a) {
  constexpr int E = D / 32;
  __shared__ float sh_o[4][D], sh_m[4], sh_l[4];
  grid_go();
  grid_wait();
  if (__syncthreads_or(*a.status != 0)) return;
  const Cache& c = a.c;
  const int h = blockIdx.x % a.heads, i = blockIdx.x / a.heads % a.S, b = blockIdx.x / a.heads / a.S;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = h / a.group;
  const int len = seen_length(c, a.lengths, b, a.status), limit = min(len, len - a.S + i + 1);
  const T* q = (const T*)a.q + b * a.q_batch + i * a.q_token + h * D + lane * E;
  float x[E], o[E], m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) {
    x[e] = to_f32<T>(q[e]) * a.scale_log2;
    o[e] = 0.f;
  }
  auto score = [&](int t, int& page) {
    page = page_of(c, b, t);
    if (page < 0) {
      atomicCAS(a.status, 0, (int)ATB_ERR_BAD_INDEX);
      page = 0;
    }
    const T* k = row_at<T, D>(c, page, 0, head, t & ((1 << c.page_shift) - 1)) + lane * E;
    float s = 0.f;
    for (int e = 0; e < E; ++e) s += x[e] * to_f32<T>(k[e]);
    return warp_sum(s);
  };
  for (int t = warp; t < limit; t += 4) {
    int page;
    const float s = score(t, page), to = fmaxf(m, s), ref = to == -INFINITY ? 0.f : to;
    const float f = exp2f(m - ref), p = exp2f(s - ref);
    const T* v = row_at<T, D>(c, page, 1, head, t & ((1 << c.page_shift) - 1)) + lane * E;
    m = to;
    l = l * f + p;
    for (int e = 0; e < E; ++e) o[e] = o[e] * f + p * to_f32<T>(v[e]);
  }
  for (int e = 0; e < E; ++e) sh_o[warp][lane * E + e] = o[e];
  sh_m[warp] = m;
  sh_l[warp] = l;
  __syncthreads();
  const float top = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3])), ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int w = 0; w < 4; ++w) sum += sh_l[w] * exp2f(sh_m[w] - ref);
  for (int d = threadIdx.x; d < D; d += 128) {
    float y = 0.f;
    for (int w = 0; w < 4; ++w) y += sh_o[w][d] * exp2f(sh_m[w] - ref);
    ((T*)a.out)[((long long)(b * a.S + i) * a.heads + h) * D + d] = from_f32<T>(sum == 0.f ? 0.f : y / sum);
  }
  if (threadIdx.x == 0 && a.lse) a.lse[((long long)b * a.heads + h) * a.S + i] = (top + log2f(sum)) * 0.69314718056f;
  if (a.partial)
    if (threadIdx.x == 0) a.partial[((long long)b * a.heads + h) * a.S + i] = top + log2f(sum);
}

// What the queries attended to, one place after another: a warp forms a key's scores again and adds their shares in the order of the
// queries.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv_weights_kernel(AttnArgs a) {
  constexpr int E = D / 32;
  grid_go();
  grid_wait();
  if (__syncthreads_or(*a.status != 0)) return;
  const Cache& c = a.c;
  const int head = blockIdx.y % c.kv_heads, b = blockIdx.y / c.kv_heads, lane = threadIdx.x & 31;
  const int len = seen_length(c, a.lengths, b, a.status);
  for (int t = blockIdx.x * 4 + (threadIdx.x >> 5); t < len; t += gridDim.x * 4) {
    const int page = page_of(c, b, t);
    if (page < 0) continue;
    const T* k = row_at<T, D>(c, page, 0, head, t & ((1 << c.page_shift) - 1)) + lane * E;
    float sum = 0.f;
    for (int i = max(0, t - len + a.S); i < a.S; ++i)
      for (int h = head * a.group; h < (head + 1) * a.group; ++h) {
        const T* q = (const T*)a.q + b * a.q_batch + i * a.q_token + h * D + lane * E;
        float s = 0.f;
        for (int e = 0; e < E; ++e) s += to_f32<T>(q[e]) * a.scale_log2 * to_f32<T>(k[e]);
        const float lse = a.partial[((long long)b * a.heads + h) * a.S + i];
        if (lse != -INFINITY) sum += exp2f(warp_sum(s) - lse);
      }
    if (lane == 0) a.weights[((long long)b * c.kv_heads + head) * a.places + t] += sum;
  }
}

// ----------------------------------------------------------------------------------
// Eviction
// ----------------------------------------------------------------------------------
struct EvictArgs {
  Cache c;
  const int* lengths;
  float* weights;
  int* out;
  int* index;                 // [units][budget + 1]
  long long places, layer_elements;
  int budget, recent, layers;
  int* status;
};
// A number whose order as an unsigned integer is that of f; both zeros alike, a NaN as -inf.
ATB_DEVICE uint32_t rank_of(float f) {
  const uint32_t u = __float_as_uint((f != f ? -INFINITY : f) + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
ATB_DEVICE int block_exclusive(int v, int* red, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  __syncthreads();
  if (lane == 31) red[w] = sum;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < warps; ++i) {
    if (i < w) before += red[i];
    all += red[i];
  }
  *total = all;
  return before + sum - v;
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv_evict_kernel(EvictArgs a) {
  __shared__ int hist[256], red[8], sh_digit, sh_left;
  grid_go();
  grid_wait();
  if (__syncthreads_or(*a.status != 0)) return;
  Cache c = a.c;
  const int head = blockIdx.x % c.kv_heads, b = blockIdx.x / c.kv_heads % c.rows, layer = blockIdx.x / c.kv_heads / c.rows;
  c.data = (T*)c.data + layer * a.layer_elements;
  const int len = seen_length(c, a.lengths, b, a.status);
  if (layer == 0 && head == 0 && threadIdx.x == 0) a.out[b] = min(a.lengths[b], a.budget);
  if (len <= a.budget) return;
  bool good = true;
  for (int i = threadIdx.x; i << c.page_shift < len; i += 256) good = good && page_of(c, b, i << c.page_shift) >= 0;
  if (__syncthreads_or(!good)) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, (int)ATB_ERR_BAD_INDEX);
    return;
  }
  float* const w = a.weights + (long long)blockIdx.x * a.places;
  int* const index = a.index + (long long)blockIdx.x * (a.budget + 1);
  const int n = len - a.recent;
  int left = a.budget - a.recent;            // of rank `rank`, so many go with the higher ones
  uint32_t rank = 0;
  if (left == 0) rank = 0xffffffffu;
  for (int shift = 24; shift >= 0 && left > 0; shift -= 8) {
    hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
      const uint32_t r = rank_of(w[i]);
      if (shift == 24 || (r >> (shift + 8)) == (rank >> (shift + 8))) atomicAdd(&hist[r >> shift & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int d = 255, k = left;
      for (; d > 0 && hist[d] < k; --d) k -= hist[d];
      sh_digit = d;
      sh_left = k;
    }
    __syncthreads();
    rank |= (uint32_t)sh_digit << shift;
    left = sh_left;
  }
  int kept = 0, ties = 0;
  for (int i0 = 0; i0 < len; i0 += 256) {
    const int i = i0 + threadIdx.x;
    const float f = i < len ? w[i] : 0.f;
    const uint32_t r = rank_of(f);
    int all_ties, all_kept;
    const bool tie = i < n && r == rank;
    const int tie_before = ties + block_exclusive(tie, red, &all_ties);
    const bool keep = i < len && (i >= n || r > rank || (tie && tie_before < left));
    const int at = kept + block_exclusive(keep, red, &all_kept);
    ties += all_ties;
    kept += all_kept;
    __syncthreads();
    if (keep) {
      index[at] = i;
      w[at] = f;
    }
  }
  __syncthreads();
  for (int i = a.budget + threadIdx.x; i < len; i += 256) w[i] = 0.f;
  constexpr int L = D / 8, EACH = 256 / L;
  const int l = threadIdx.x % L, mask = (1 << c.page_shift) - 1;
  for (int j0 = 0; j0 < a.budget; j0 += EACH) {
    const int j = j0 + threadIdx.x / L;
    uint4 x[2];
    if (j < a.budget) {
      const int src = index[j], page = page_of(c, b, src);
      for (int i = 0; i < 2; ++i) x[i] = *reinterpret_cast<const uint4*>(row_at<T, D>(c, page, i, head, src & mask) + l * 8);
    }
    __syncthreads();
    if (j < a.budget) {
      const int page = page_of(c, b, j);
      for (int i = 0; i < 2; ++i) *reinterpret_cast<uint4*>(row_at<T, D>(c, page, i, head, j & mask) + l * 8) = x[i];
    }
    __syncthreads();
  }
}

Cache cache_of(void* data, const void* table, long long table_stride, int rows, int width, int pages, int kv_heads, int page_shift) {
  return Cache{{(const int*)table, table_stride, rows, width, pages, kv_heads, page_shift}, data};
}

template <typename T, int D>
int launch_append(const void* qkv, void* q, void* k, const Cache& c, const void* seq, const void* pos, const void* angles,
                  const void* cosT, const void* sinT, int positions, int tokens, int n_q, long long stride, cudaStream_t st, int* status) {
  const int each = SMALL / (D / 16), heads = n_q + 2 * c.kv_heads, blocks = (heads + each - 1) / each;
  if (blocks > 65535) return -2;
  return launched(launch_after(kv_append_kernel<T, D, 1>, dim3(tokens, blocks), SMALL, 0, st, 1, (const T*)qkv, (T*)q, (T*)k, c,
                               (const int*)seq, (const int*)pos, (const int*)angles, (const float*)cosT, (const float*)sinT, positions,
                               n_q, stride, status));
}

template <typename T, int D>
int launch_attention(const AttnArgs& a, cudaStream_t st) {
  const long long blocks = (long long)a.c.rows * a.S * a.heads;
  if (blocks > 0x7fffffffLL || (long long)a.c.rows * a.c.kv_heads > 65535) return -2;
  const int rc = launched(launch_after(kv_attention_kernel<T, D>, dim3((unsigned)blocks), 128, 0, st, 1, a));
  if (rc != 0 || !a.weights) return rc;
  return launched(launch_after(kv_weights_kernel<T, D>, dim3(64, a.c.rows * a.c.kv_heads), 128, 0, st, 1, a));
}

template <typename T, int D>
int launch_evict(const EvictArgs& a, cudaStream_t st) {
  const long long units = (long long)a.layers * a.c.rows * a.c.kv_heads;
  if (units > 0x7fffffffLL) return -2;
  return launched(launch_after(kv_evict_kernel<T, D>, dim3((unsigned)units), 256, 0, st, 1, a));
}
}  // namespace

#define ATB_KV_TYPES(F)                                  \
  if (dtype == 0 && head_dim == 64) F(__nv_bfloat16, 64);   \
  if (dtype == 0 && head_dim == 128) F(__nv_bfloat16, 128); \
  if (dtype == 1 && head_dim == 64) F(__half, 64);          \
  if (dtype == 1 && head_dim == 128) F(__half, 128);

extern "C" int atb_kv_append(const void* qkv, void* q, void* k, void* data, const void* table, const void* seq, const void* pos,
                             const void* angles, const void* cosT, const void* sinT, int positions, int tokens, int n_q,
                             int kv_heads, int head_dim, int page_shift, int pages, int rows, int width, long long table_stride,
                             long long token_stride, int dtype, void* stream, void* status) {
  if (tokens <= 0) return 0;
  const Cache c = cache_of(data, table, table_stride, rows, width, pages, kv_heads, page_shift);
#define APPEND(T, D)                                                                                                         \
  return launch_append<T, D>(qkv, q, k, c, seq, pos, angles, cosT, sinT, positions, tokens, n_q, token_stride, (cudaStream_t)stream, \
                             (int*)status)
  ATB_KV_TYPES(APPEND)
#undef APPEND
  return -1;
}

// Floats of the workspace of atb_kv_attention.
extern "C" long long atb_kv_attention_scratch(int rows, int heads, int kv_heads, int S, int head_dim, int places, int weighed) {
  return weighed ? (long long)rows * heads * S : 0;
}

extern "C" int atb_kv_attention(const void* q, void* out, void* lse, void* data, const void* table, const void* lengths, void* weights,
                                void* partial, int S, int heads, int kv_heads, int head_dim, int page_shift, int pages, int rows,
                                int width, long long table_stride, long long places, long long q_batch, long long q_token, float scale,
                                int dtype, void* stream, void* status) {
  if (rows <= 0 || S <= 0) return 0;
  AttnArgs a;
  a.c = cache_of(data, table, table_stride, rows, width, pages, kv_heads, page_shift);
  a.lengths = (const int*)lengths;
  a.q = q;
  a.out = out;
  a.lse = (float*)lse;
  a.weights = (float*)weights;
  a.partial = (float*)partial;
  a.places = places;
  a.q_batch = q_batch;
  a.q_token = q_token;
  a.S = S;
  a.heads = heads;
  a.group = heads / kv_heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = (int*)status;
#define ATTN(T, D) return launch_attention<T, D>(a, (cudaStream_t)stream)
  ATB_KV_TYPES(ATTN)
#undef ATTN
  return -1;
}

extern "C" int atb_kv_evict(void* data, const void* table, const void* lengths, void* weights, void* out, void* index, int layers,
                            int kv_heads, int head_dim, int page_shift, int pages, int rows, int width, long long table_stride,
                            long long places, int budget, int recent, void* stream, void* status) {
  if (rows <= 0) return 0;
  EvictArgs a;
  a.c = cache_of(data, table, table_stride, rows, width, pages, kv_heads, page_shift);
  a.lengths = (const int*)lengths;
  a.weights = (float*)weights;
  a.out = (int*)out;
  a.index = (int*)index;
  a.places = places;
  a.layer_elements = ((long long)pages * 2 * kv_heads << page_shift) * head_dim;
  a.budget = budget;
  a.recent = recent;
  a.layers = layers;
  a.status = (int*)status;
  if (head_dim == 64) return launch_evict<__half, 64>(a, (cudaStream_t)stream);      // (16 bits are moved as they are)
  if (head_dim == 128) return launch_evict<__half, 128>(a, (cudaStream_t)stream);
  return -1;
}
