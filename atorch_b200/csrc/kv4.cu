// Paged key/value cache in 4 bits: append with rotation, reading back, attention of the newest tokens.
//
// One layer's cache:
//   codes  uint8 [pages][2][kv heads][page size][D / 2]    0: keys, 1: values; byte i: dim 2i low, dim 2i + 1 high
//   scales bf16  [pages][kv heads][page size][4]           scale and minimum of the key, scale and minimum of the value
// A value is code * scale + minimum, one scale and minimum per token, head and tensor: (D + 8) bytes a token and head where
// bf16 keeps 4 D. Sequence b's token p lies in page table[b][p / page size], place p % page size.
#include "common.cuh"

namespace {
using namespace atb;

struct Cache {
  uint8_t* codes;
  __nv_bfloat16* scales;
  const int* table;
  long long table_stride;
  int rows, width;       // sequences, pages a sequence may have
  int pages, kv_heads, page_shift;
};

// Page of token p of sequence b, or -1 where the table or the sequence does not have it.
ATB_DEVICE int page_of(const Cache& c, int b, int p) {
  const int i = p >> c.page_shift;
  if (b < 0 || b >= c.rows || i >= c.width) return -1;
  const int page = c.table[b * c.table_stride + i];
  return page < 0 || page >= c.pages ? -1 : page;
}
template <int D>
ATB_DEVICE uint8_t* codes_at(const Cache& c, int page, int which, int head, int slot) {
  return c.codes + (((((long long)page * 2 + which) * c.kv_heads + head) << c.page_shift) + slot) * (D / 2);
}
ATB_DEVICE __nv_bfloat16* scales_at(const Cache& c, int page, int head, int slot) {
  return c.scales + ((((long long)page * c.kv_heads + head) << c.page_shift) + slot) * 4;
}

template <typename T>
ATB_DEVICE void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(h[i]);
  }
}
template <typename T>
ATB_DEVICE void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint4 u;
    T* h = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(x[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}
// minimum and maximum that keep a NaN: a token with one stands for NaN, as its values would
ATB_DEVICE float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
ATB_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A head of a token is D / 16 lanes: each has 8 dims of the first half and the 8 of the second half that they turn with.
// Rotation and codes are computed by separately rounded fp32 operations (no fused multiply-add, true division), so that the
// codes are those of the formula evaluated operation by operation, and do not depend on how a compiler contracts it. The scale
// is rounded to bf16 before the codes are taken: the code is the nearest one of the scale that is kept.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const T* qkv, T* q_out, Cache c, const int* seq, const int* pos,
                                                         const float* cosT, const float* sinT, int positions,
                                                         long long units, int n_q, long long token_stride, int* status) {
  grid_go();
  grid_wait();
  constexpr int L = D / 16, HALF = D / 2;
  const int heads = n_q + 2 * c.kv_heads;
  const long long thread = blockIdx.x * 256ll + threadIdx.x;
  const long long unit = thread / L;
  const int l = (int)(thread % L);
  const bool failed = warp_uniform(*status) != 0;       // one answer for the lanes of a head; asked by all lanes
  const bool live = unit < units && !failed;
  const long long t = live ? unit / heads : 0;
  const int h = live ? (int)(unit - t * heads) : 0;
  float a[8], b[8];
  int p = -1, page = -1;
  if (live) {
    const T* src = qkv + t * token_stride + (long long)h * D + l * 8;
    load8<T>(src, a);
    load8<T>(src + HALF, b);
    p = pos[t];
    if (p >= 0) {
      page = page_of(c, seq ? seq[t] : (int)t, p);
      if (page < 0 || (cosT && p >= positions)) {
        atomicCAS(status, 0, (int)ATB_ERR_BAD_INDEX);
        page = -1;
        p = -1;
      }
    }
  }
  if (cosT && p >= 0 && h < n_q + c.kv_heads) {
    float cs[8], sn[8];
    load8<float>(cosT + (long long)p * HALF + l * 8, cs);
    load8<float>(sinT + (long long)p * HALF + l * 8, sn);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a[i], y = b[i];
      a[i] = __fsub_rn(__fmul_rn(x, cs[i]), __fmul_rn(y, sn[i]));
      b[i] = __fadd_rn(__fmul_rn(y, cs[i]), __fmul_rn(x, sn[i]));
    }
  }
  if (live && h < n_q) {
    T* dst = q_out + (t * n_q + h) * D + l * 8;
    store8<T>(dst, a);
    store8<T>(dst + HALF, b);
  }
  float lo = 0.f, hi = 0.f;
  if (live) {
    lo = min_nan(a[0], b[0]);
    hi = max_nan(a[0], b[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      lo = min_nan(lo, min_nan(a[i], b[i]));
      hi = max_nan(hi, max_nan(a[i], b[i]));
    }
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (!live || h < n_q || page < 0) return;
  const __nv_bfloat16 scale = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f)), low = __float2bfloat16_rn(lo);
  const float s = __bfloat162float(scale), m = __bfloat162float(low);
  uint32_t w[2] = {0u, 0u};
  if (s > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(a[i], m), s)), 0.f), 15.f);
      const float v = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(b[i], m), s)), 0.f), 15.f);
      w[0] |= (uint32_t)u << (4 * i);
      w[1] |= (uint32_t)v << (4 * i);
    }
  }
  const int which = h >= n_q + c.kv_heads, head = h - n_q - (which ? c.kv_heads : 0), slot = p & ((1 << c.page_shift) - 1);
  uint8_t* dst = codes_at<D>(c, page, which, head, slot) + l * 4;
  *reinterpret_cast<uint32_t*>(dst) = w[0];
  *reinterpret_cast<uint32_t*>(dst + HALF / 2) = w[1];
  if (l == 0) {
    const __nv_bfloat162 pair = __halves2bfloat162(scale, low);
    reinterpret_cast<__nv_bfloat162*>(scales_at(c, page, head, slot))[which] = pair;
  }
}

// What the cache stands for at given tokens: a lane turns 8 codes of the keys and of the values into two 16-byte pieces.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(T* k, T* v, Cache c, const int* seq, const int* pos, long long units,
                                                       int* status) {
  grid_go();
  grid_wait();
  constexpr int L = D / 8;
  const long long thread = blockIdx.x * 256ll + threadIdx.x;
  const long long unit = thread / L;
  const int l = (int)(thread % L);
  if (unit >= units || *status != 0) return;
  const long long t = unit / c.kv_heads;
  const int h = (int)(unit - t * c.kv_heads), p = pos[t];
  float x[2][8] = {};
  if (p >= 0) {
    const int page = page_of(c, seq ? seq[t] : (int)t, p), slot = p & ((1 << c.page_shift) - 1);
    if (page < 0) {
      atomicCAS(status, 0, (int)ATB_ERR_BAD_INDEX);
    } else {
      const uint2 sc = *reinterpret_cast<const uint2*>(scales_at(c, page, h, slot));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes_at<D>(c, page, i, h, slot) + l * 4);
        const float2 f = unpack_bf16x2(i ? sc.y : sc.x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = (float)((w >> (4 * e)) & 15u) * f.x + f.y;
      }
    }
  }
  store8<T>(k + unit * D + l * 8, x[0]);
  store8<T>(v + unit * D + l * 8, x[1]);
}

// ----------------------------------------------------------------------------------
// Attention
// ----------------------------------------------------------------------------------
// Query i of sequence b's S newest tokens sees its keys j < lengths[b] - S + i + 1. The g query heads of a key/value head times
// the S tokens are the columns of one matrix product: n = i g + h, in tiles of 8.
//
// The sequences are cut into chunks of equal length, as many as fill the GPU, by every block for itself from the lengths on the
// device (they need not be known on the host); a block takes chunks of a head until there are none left. Sequences of one chunk
// are finished in place, the others leave sums, maximum and denominator per chunk, which a second kernel joins in their order.
constexpr int WARPS = 4, MIN_CHUNK = 64, TILE = 16;

struct Plan {
  int chunk;             // tokens, a multiple of MIN_CHUNK
  long long chunks;      // of all sequences
};
ATB_DEVICE int seen_length(const Cache& c, const int* lengths, int b, int* status) {
  const int n = lengths[b], most = c.width << c.page_shift;
  if (n > most) atomicCAS(status, 0, (int)ATB_ERR_BAD_INDEX);
  return max(0, min(n, most));
}
ATB_DEVICE int chunks_of(int n, int chunk) { return max(1, (n + chunk - 1) / chunk); }
ATB_DEVICE long long warp_sum_ll(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// `per`: blocks that a chunk occupies (heads x column tiles); `ctas`: blocks that the GPU is to be filled with
ATB_DEVICE Plan make_plan(const Cache& c, const int* lengths, int per, int ctas, int* status) {
  const int lane = threadIdx.x & 31;
  long long total = 0;
  for (int b = lane; b < c.rows; b += 32) total += seen_length(c, lengths, b, status);
  total = warp_sum_ll(total);
  const long long want = (total * per + ctas - 1) / ctas;
  Plan p;
  p.chunk = (int)max((long long)MIN_CHUNK, (want + MIN_CHUNK - 1) / MIN_CHUNK * MIN_CHUNK);
  long long n = 0;
  for (int b = lane; b < c.rows; b += 32) n += chunks_of(seen_length(c, lengths, b, status), p.chunk);
  p.chunks = warp_sum_ll(n);
  return p;
}
// Sequence b of chunk number `w`, the chunk's place in it, and the number of the first partial result of b (only sequences of
// several chunks have any). Computed by a whole warp.
ATB_DEVICE void find_chunk(const Cache& c, const int* lengths, const Plan& p, long long w, int& b, int& place, int& of,
                           int& len, long long& partial, int* status) {
  const int lane = threadIdx.x & 31;
  long long before = 0, before_partial = 0;
  for (int b0 = 0; b0 < c.rows; b0 += 32) {
    const int n = b0 + lane < c.rows ? seen_length(c, lengths, b0 + lane, status) : 0;
    const int k = b0 + lane < c.rows ? chunks_of(n, p.chunk) : 0;
    int sum = k, sum_partial = k > 1 ? k : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o), y = __shfl_up_sync(0xffffffffu, sum_partial, o);
      if (lane >= o) {
        sum += x;
        sum_partial += y;
      }
    }
    const unsigned hit = __ballot_sync(0xffffffffu, w < before + sum);
    if (hit) {
      const int src = __ffs(hit) - 1;
      b = b0 + src;
      of = __shfl_sync(0xffffffffu, k, src);
      len = __shfl_sync(0xffffffffu, n, src);
      place = (int)(w - before) - __shfl_sync(0xffffffffu, sum - k, src);
      partial = before_partial + __shfl_sync(0xffffffffu, sum_partial, src) - (of > 1 ? of : 0);
      return;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
    before_partial += __shfl_sync(0xffffffffu, sum_partial, 31);
  }
  b = -1;
}

ATB_DEVICE void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
ATB_DEVICE uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
ATB_DEVICE uint32_t pack_f16x2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
ATB_DEVICE float pow2(int e) { return __int_as_float((e + 127) << 23); }     // -126 <= e <= 127

template <int WORDS>
struct Words {
  uint32_t w[WORDS];
};
template <int WORDS>
ATB_DEVICE Words<WORDS> load_words(const void* p) {
  Words<WORDS> r;
  if constexpr (WORDS == 1) r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  if constexpr (WORDS == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    r.w[0] = u.x; r.w[1] = u.y;
  }
  if constexpr (WORDS >= 4) {
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[i];
      r.w[4 * i] = u.x; r.w[4 * i + 1] = u.y; r.w[4 * i + 2] = u.z; r.w[4 * i + 3] = u.w;
    }
  }
  return r;
}

struct AttnArgs {
  Cache c;
  const int* lengths;
  const void* q;
  void* out;
  float* lse;                 // [rows][heads][S] or nullptr
  float* partial;             // sums [..][D], then maximum and denominator [..][2]
  long long partial_rows;
  long long q_batch, q_token; // strides of q, elements
  int S, heads, group;
  float scale_log2;           // softmax scale * log2(e)
  int ctas;
  int* status;
};

// Both products run on the warp's matrix instruction (16 x 8 x 16, fp16, fp32 sums) with the codes as its 16-row operand. A
// code needs no conversion: its 4 bits, alone in the low bits of a half, are the fp16 number code * 2^-24, and four places
// further up code * 2^-20; so eight codes cost four ANDs and a shift. The other operand takes the powers of two and everything
// else that a value has:
//   s[t, n]  = ks[t] (q[n] . code[t]) + km[t] sum(q[n])        o[d, n] = sum_t (p[t, n] vs[t]) code[t, d] + sum_t p[t, n] vm[t]
// q is scaled by a power of two to at most 2^15 before it is rounded to fp16 (bf16 and fp16 values stay exact down to 2^-29 of
// the largest), p vs by 2^(15 - e) with e the largest exponent of a value's scale so far, as the maximum of a softmax runs:
// 11 bits of it are kept, which is what the products with 4-bit codes can use. Sums, maxima and denominators are fp32.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(WARPS * 32) kv4_attention_kernel(AttnArgs a) {
  constexpr int KW = D / 32, VW = D / 64, COLS = 8 * NT, MT = D / 16;
  __shared__ float sh_o[WARPS][COLS][D + 4];
  __shared__ float sh_m[WARPS][COLS], sh_l[WARPS][COLS];
  grid_go();
  grid_wait();
  if (__syncthreads_or(threadIdx.x == 0 && *a.status != 0)) return;    // one answer for the block: others may fail meanwhile
  const Cache& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, q4 = lane & 3;
  const int columns = a.S * a.group, tiles = (columns + COLS - 1) / COLS, per = tiles * c.kv_heads;
  const Plan plan = make_plan(c, a.lengths, per, a.ctas, a.status);
  const int page_mask = (1 << c.page_shift) - 1;

  for (long long item = blockIdx.x; item < plan.chunks * per; item += gridDim.x) {
    const long long w = item / per;
    const int head = (int)(item - w * per) % c.kv_heads, tile = (int)(item - w * per) / c.kv_heads;
    int b, place, of, len;
    long long first_partial;
    find_chunk(c, a.lengths, plan, w, b, place, of, len, first_partial, a.status);
    const int t_begin = place * plan.chunk, t_end = min(len, t_begin + plan.chunk);

    // queries: column 8 j + r, this lane's quarter of the dims; class-1 dims (odd places of a word) carry 2^-4
    uint32_t qf[NT][KW][4];
    float cs[NT][2], bs[NT][2];      // factors of the products and sum(q) of the columns 8 j + 2 q4 + {0, 1}
    int limit[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = tile * COLS + 8 * j + r;
      const bool live = n < columns;
      const int i = live ? n / a.group : 0, h = live ? n - i * a.group : 0;
      const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_batch + i * a.q_token +
                   (long long)(head * a.group + h) * D + q4 * (D / 4);
      float x[KW][8], top = 0.f, sum = 0.f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        if (live) {
          load8<T>(q + 8 * k, x[k]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          top = fmaxf(top, fabsf(x[k][e]));
          sum += x[k][e];
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
      }
      const int e = top > 0.f ? min(max((__float_as_int(top) >> 23) - 127, -100), 100) : 0;   // top < 2^(e + 1)
      const float up = pow2(14 - e);
#pragma unroll
      for (int k = 0; k < KW; ++k)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float f = p & 1 ? up * 0.0625f : up;
          qf[j][k][p] = pack_f16x2(x[k][p] * f, x[k][p + 4] * f);
        }
      const float back = pow2(10 + e) * a.scale_log2;      // 2^24 / 2^(14 - e)
      sum *= a.scale_log2;
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        cs[j][o] = __shfl_sync(0xffffffffu, back, (2 * q4 + o) * 4);
        bs[j][o] = __shfl_sync(0xffffffffu, sum, (2 * q4 + o) * 4);
        const int col = tile * COLS + 8 * j + 2 * q4 + o;
        limit[j][o] = min(t_end, len - a.S + col / a.group + 1);
      }
    }

    float o_acc[NT][MT][4], m[NT][2], l[NT][2], z[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o_acc[j][i][e] = 0.f;
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        m[j][o] = -INFINITY;
        l[j][o] = z[j][o] = 0.f;
      }
    }
    int top_e = 16;        // exponent field of the largest value scale so far

    for (int t0 = t_begin + warp * TILE; t0 < t_end; t0 += WARPS * TILE) {
      int page = c.table[b * c.table_stride + (t0 >> c.page_shift)];
      if (page < 0 || page >= c.pages) {
        if (lane == 0) atomicCAS(a.status, 0, (int)ATB_ERR_BAD_INDEX);
        page = 0;
      }
      const int slot = t0 & page_mask;
      Words<KW> kc[2];
      Words<VW> vc[4];
      uint2 sc[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kc[i] = load_words<KW>(codes_at<D>(c, page, 0, head, slot + r + 8 * i) + q4 * (KW * 4));
        sc[i] = *reinterpret_cast<const uint2*>(scales_at(c, page, head, slot + r + 8 * i));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        vc[i] = load_words<VW>(codes_at<D>(c, page, 1, head, slot + 2 * q4 + (i & 1) + 8 * (i >> 1)) + r * (VW * 4));

      float s[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const uint32_t x = kc[0].w[k], y = kc[1].w[k], xs = x >> 8, ys = y >> 8;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma_f16(s[j], x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, qf[j][k][0], qf[j][k][1]);
          mma_f16(s[j], xs & 0x000F000Fu, ys & 0x000F000Fu, xs & 0x00F000F0u, ys & 0x00F000F0u, qf[j][k][2], qf[j][k][3]);
        }
      }

      float2 ks[2], vs[2];
      int e_new = top_e;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool in = t0 + r + 8 * i < t_end;       // places behind the last token hold anything
        ks[i] = unpack_bf16x2(in ? sc[i].x : 0u);
        vs[i] = unpack_bf16x2(in ? sc[i].y : 0u);
        const int e = (__float_as_int(vs[i].x) >> 23) & 255;
        e_new = max(e_new, e == 255 ? 0 : e);         // an infinity is not for the queries that do not see it
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) e_new = max(e_new, __shfl_xor_sync(0xffffffffu, e_new, o));

      float m_new[NT][2];
      bool moved = e_new != top_e;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          m_new[j][o] = m[j][o];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float& x = s[j][2 * i + o];
            x = t0 + r + 8 * i < limit[j][o] ? fmaf(ks[i].x, x * cs[j][o], ks[i].y * bs[j][o]) : -INFINITY;
            m_new[j][o] = fmaxf(m_new[j][o], x);
          }
#pragma unroll
          for (int k = 4; k < 32; k <<= 1) m_new[j][o] = fmaxf(m_new[j][o], __shfl_xor_sync(0xffffffffu, m_new[j][o], k));
          moved = moved || m_new[j][o] != m[j][o];
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
        const float down = __int_as_float((127 + max(top_e - e_new, -126)) << 23);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float f[2];
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            f[o] = m[j][o] == -INFINITY ? 0.f : fast_exp2(m[j][o] - m_new[j][o]);
            l[j][o] *= f[o];
            z[j][o] *= f[o];
            m[j][o] = m_new[j][o];
            f[o] *= down;
          }
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o_acc[j][i][e] *= f[e & 1];
        }
        top_e = e_new;
      }
      const float up = __int_as_float((268 - top_e) << 23);      // 2^15 / 2^(exponent + 1)
      uint32_t pf[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float ref[2] = {m[j][0] == -INFINITY ? 0.f : m[j][0], m[j][1] == -INFINITY ? 0.f : m[j][1]};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float pv[2];
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const bool seen = t0 + r + 8 * i < limit[j][o];
            const float p = fast_exp2(s[j][2 * i + o] - ref[o]);
            l[j][o] += p;
            z[j][o] += seen ? p * vs[i].y : 0.f;
            pv[o] = seen ? p * (vs[i].x * up) : 0.f;
          }
          pf[j][i] = transpose_8x8(pack_f16x2(pv[0], pv[1]));
        }
      }
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        // words of two neighbouring tokens side by side: places 0 to 3 of both, then 4 to 7
        const uint32_t lo0 = __byte_perm(vc[0].w[k], vc[1].w[k], 0x5410), hi0 = __byte_perm(vc[0].w[k], vc[1].w[k], 0x7632);
        const uint32_t lo1 = __byte_perm(vc[2].w[k], vc[3].w[k], 0x5410), hi1 = __byte_perm(vc[2].w[k], vc[3].w[k], 0x7632);
        const uint32_t x[4] = {lo0, lo0 >> 8, hi0, hi0 >> 8}, y[4] = {lo1, lo1 >> 8, hi1, hi1 >> 8};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
            mma_f16(o_acc[j][4 * k + i], x[i] & 0x000F000Fu, x[i] & 0x00F000F0u, y[i] & 0x000F000Fu, y[i] & 0x00F000F0u,
                    pf[j][0], pf[j][1]);
      }
    }

    // the warps' sums, in their order
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int o = 0; o < 2; ++o) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
          l[j][o] += __shfl_xor_sync(0xffffffffu, l[j][o], k);
          z[j][o] += __shfl_xor_sync(0xffffffffu, z[j][o], k);
        }
        const int col = 8 * j + 2 * q4 + o;
        if (r == 0) {
          sh_m[warp][col] = m[j][o];
          sh_l[warp][col] = l[j][o];
        }
        const float f = pow2(min(top_e - 121, 127));           // 2^20 / (2^15 / 2^(exponent + 1)) of the odd places
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          sh_o[warp][col][r * (D / 8) + 2 * i] = o_acc[j][i][o] * (16.f * f) + z[j][o];
          sh_o[warp][col][r * (D / 8) + 2 * i + 1] = o_acc[j][i][2 + o] * f + z[j][o];
        }
      }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < COLS * (D / 4); x += WARPS * 32) {
      const int col = x / (D / 4), d = (x - col * (D / 4)) * 4, n = tile * COLS + col;
      if (n >= columns) continue;
      float top = sh_m[0][col];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) top = fmaxf(top, sh_m[k][col]);
      float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float f = sh_m[k][col] == -INFINITY ? (sh_l[k][col] == 0.f ? 0.f : 1.f) : fast_exp2(sh_m[k][col] - top);
        sum += f * sh_l[k][col];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += f * sh_o[k][col][d + e];
      }
      const int i = n / a.group, h = head * a.group + n - i * a.group;
      if (of > 1) {
        const long long row = (first_partial + place) * ((long long)a.heads * a.S) + (long long)h * a.S + i;
        *reinterpret_cast<float4*>(a.partial + row * D + d) = make_float4(o[0], o[1], o[2], o[3]);
        if (d == 0) *reinterpret_cast<float2*>(a.partial + a.partial_rows * D + row * 2) = make_float2(top, sum);
      } else {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(o[e] * inv);
        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + (((long long)b * a.S + i) * a.heads + h) * D + d) =
            *reinterpret_cast<const uint2*>(y);
        if (d == 0 && a.lse) a.lse[((long long)b * a.heads + h) * a.S + i] = (top + log2f(sum)) * 0.69314718056f;
      }
    }
  }
}

// Sequences of several chunks: one warp per row of the output.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_join_kernel(AttnArgs a, int per) {
  grid_go();
  grid_wait();
  if (warp_uniform(*a.status) != 0) return;
  const int lane = threadIdx.x & 31;
  const long long row = blockIdx.x * 4ll + (threadIdx.x >> 5);      // (b, h, i)
  if (row >= (long long)a.c.rows * a.heads * a.S) return;
  const int b = (int)(row / ((long long)a.heads * a.S)), hi = (int)(row - (long long)b * a.heads * a.S);
  const Plan plan = make_plan(a.c, a.lengths, per, a.ctas, a.status);
  const int of = chunks_of(seen_length(a.c, a.lengths, b, a.status), plan.chunk);
  if (of == 1) return;
  long long first = 0;
  for (int x = lane; x < b; x += 32) {
    const int k = chunks_of(seen_length(a.c, a.lengths, x, a.status), plan.chunk);
    first += k > 1 ? k : 0;
  }
  first = warp_sum_ll(first);
  const float* stats = a.partial + a.partial_rows * D;
  const long long step = (long long)a.heads * a.S, at = first * step + hi;
  float top = -INFINITY;
  for (int k = lane; k < of; k += 32) top = fmaxf(top, stats[(at + k * step) * 2]);
  top = warp_max(top);
  float sum = 0.f, o[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int k = 0; k < of; ++k) {
    const float2 ml = *reinterpret_cast<const float2*>(stats + (at + k * step) * 2);
    const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - top);
    sum += f * ml.y;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] += f * a.partial[(at + k * step) * D + lane + 32 * e];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int h = hi / a.S, i = hi - h * a.S;
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
    reinterpret_cast<T*>(a.out)[(((long long)b * a.S + i) * a.heads + h) * D + lane + 32 * e] = from_f32<T>(o[e] * inv);
  if (lane == 0 && a.lse) a.lse[row] = (top + log2f(sum)) * 0.69314718056f;
}

Cache cache_of(void* codes, void* scales, const void* table, long long table_stride, int rows, int width, int pages,
               int kv_heads, int page_shift) {
  return Cache{(uint8_t*)codes, (__nv_bfloat16*)scales, (const int*)table, table_stride, rows, width, pages, kv_heads, page_shift};
}

template <typename T, int D>
int launch_append(const void* qkv, void* q, const Cache& c, const void* seq, const void* pos, const void* cosT, const void* sinT,
                  int positions, int tokens, int n_q, long long stride, cudaStream_t st, int* status) {
  const long long units = (long long)tokens * (n_q + 2 * c.kv_heads), blocks = (units * (D / 16) + 255) / 256;
  if (blocks > 0x7fffffffLL) return -2;
  return launch_after(kv4_append_kernel<T, D>, dim3((unsigned)blocks), 256, 0, st, 1, (const T*)qkv, (T*)q, c, (const int*)seq,
                      (const int*)pos, (const float*)cosT, (const float*)sinT, positions, units, n_q, stride,
                      status) == cudaSuccess ? 0 : -5;
}
template <typename T, int D>
int launch_read(void* k, void* v, const Cache& c, const void* seq, const void* pos, int tokens, cudaStream_t st, int* status) {
  const long long units = (long long)tokens * c.kv_heads, blocks = (units * (D / 8) + 255) / 256;
  if (blocks > 0x7fffffffLL) return -2;
  return launch_after(kv4_read_kernel<T, D>, dim3((unsigned)blocks), 256, 0, st, 1, (T*)k, (T*)v, c, (const int*)seq,
                      (const int*)pos, units, status) == cudaSuccess ? 0 : -5;
}

constexpr int CTAS = 148 * 4;

template <typename T, int D, int NT>
int launch_attention(const AttnArgs& a, bool join, cudaStream_t st) {
  const int tiles = (a.S * a.group + 8 * NT - 1) / (8 * NT), per = tiles * a.c.kv_heads;
  // no more blocks than chunks there can be
  const long long of = (((long long)a.c.width << a.c.page_shift) + MIN_CHUNK - 1) / MIN_CHUNK;
  const long long most = (of > 1 ? of : 1) * a.c.rows * per;
  const unsigned grid = (unsigned)(most < CTAS ? most : (long long)CTAS);
  if (launch_after(kv4_attention_kernel<T, D, NT>, dim3(grid), WARPS * 32, 0, st, 1, a) != cudaSuccess) return -5;
  if (!join) return 0;
  const long long rows = (long long)a.c.rows * a.heads * a.S, blocks = (rows + 3) / 4;
  if (blocks > 0x7fffffffLL) return -2;
  return launch_after(kv4_join_kernel<T, D>, dim3((unsigned)blocks), 128, 0, st, 1, a, per) == cudaSuccess ? 0 : -5;
}
}  // namespace

extern "C" int atb_kv4_append(const void* qkv, void* q, void* codes, void* scales, const void* table, const void* seq,
                              const void* pos, const void* cosT, const void* sinT, int positions, int tokens, int n_q,
                              int kv_heads, int head_dim, int page_shift, int pages, int rows, int width,
                              long long table_stride, long long token_stride, int dtype, void* stream, void* status) {
  if (tokens <= 0) return 0;
  const Cache c = cache_of(codes, scales, table, table_stride, rows, width, pages, kv_heads, page_shift);
#define APPEND(T, D)                                                                                                 \
  return launch_append<T, D>(qkv, q, c, seq, pos, cosT, sinT, positions, tokens, n_q, token_stride, (cudaStream_t)stream, \
                             (int*)status)
#define DIMS(F, T)                  \
  if (head_dim == 64) F(T, 64);     \
  if (head_dim == 128) F(T, 128);
  if (dtype == 0) { DIMS(APPEND, __nv_bfloat16) }
  if (dtype == 1) { DIMS(APPEND, __half) }
  if (dtype == 2) { DIMS(APPEND, float) }
#undef APPEND
  return -1;
}

extern "C" int atb_kv4_read(void* k, void* v, void* codes, void* scales, const void* table, const void* seq, const void* pos,
                            int tokens, int kv_heads, int head_dim, int page_shift, int pages, int rows, int width,
                            long long table_stride, int dtype, void* stream, void* status) {
  if (tokens <= 0) return 0;
  const Cache c = cache_of(codes, scales, table, table_stride, rows, width, pages, kv_heads, page_shift);
#define READ(T, D) return launch_read<T, D>(k, v, c, seq, pos, tokens, (cudaStream_t)stream, (int*)status)
  if (dtype == 0) { DIMS(READ, __nv_bfloat16) }
  if (dtype == 1) { DIMS(READ, __half) }
  if (dtype == 2) { DIMS(READ, float) }
#undef READ
#undef DIMS
  return -1;
}

// Rows of the workspace of partial results ((D + 2) floats each): a sequence of several chunks has fewer than twice as many as
// its length in chunks, and all lengths together make no more chunks than the blocks that the GPU is filled with.
extern "C" int atb_kv4_partial_rows(int heads, int kv_heads, int S) {
  const int columns = S * (heads / kv_heads), nt = columns > 8 ? 2 : 1, per = (columns + 8 * nt - 1) / (8 * nt) * kv_heads;
  return (2 * (CTAS / per) + 2) * heads * S;
}

extern "C" int atb_kv4_attention(const void* q, void* out, void* lse, void* codes, void* scales, const void* table,
                                 const void* lengths, void* partial, int partial_rows, int S, int heads, int kv_heads,
                                 int head_dim, int page_shift, int pages, int rows, int width, long long table_stride,
                                 long long q_batch, long long q_token, float scale, int dtype, void* stream, void* status) {
  if (rows <= 0 || S <= 0) return 0;
  AttnArgs a;
  a.c = cache_of(codes, scales, table, table_stride, rows, width, pages, kv_heads, page_shift);
  a.lengths = (const int*)lengths;
  a.q = q;
  a.out = out;
  a.lse = (float*)lse;
  a.partial = (float*)partial;
  a.partial_rows = partial_rows;
  a.q_batch = q_batch;
  a.q_token = q_token;
  a.S = S;
  a.heads = heads;
  a.group = heads / kv_heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.ctas = CTAS;
  a.status = (int*)status;
  const bool join = partial != nullptr;
  if (!join && ((long long)width << page_shift) > MIN_CHUNK) return -1;
  const bool two = S * a.group > 8;
#define ATTN(T, D) \
  return two ? launch_attention<T, D, 2>(a, join, (cudaStream_t)stream) : launch_attention<T, D, 1>(a, join, (cudaStream_t)stream)
  if (dtype == 0 && head_dim == 64) ATTN(__nv_bfloat16, 64);
  if (dtype == 0 && head_dim == 128) ATTN(__nv_bfloat16, 128);
  if (dtype == 1 && head_dim == 64) ATTN(__half, 64);
  if (dtype == 1 && head_dim == 128) ATTN(__half, 128);
#undef ATTN
  return -1;
}
