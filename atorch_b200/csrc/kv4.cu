// Paged key/value cache in 4 bits: append with rotation, reading back, attention of the newest tokens.
//
// One layer's cache:
//   codes  uint8 [pages][2][kv heads][page size][D / 2]    0: keys, 1: values; byte i: dim 2i low, dim 2i + 1 high
//   scales bf16  [pages][kv heads][page size][4]           scale and minimum of the key, scale and minimum of the value
// A value is code * scale + minimum, one scale and minimum per token, head and tensor: (D + 8) bytes a token and head where
// bf16 keeps 4 D.
#include <atomic>
#include <type_traits>
#include "paged.cuh"

namespace {
using namespace atb;

struct Cache : Paging {
  uint8_t* codes;
  __nv_bfloat16* scales;
};

template <int D>
ATB_DEVICE uint8_t* codes_at(const Cache& c, int page, int which, int head, int slot) {
  return c.codes + (((((long long)page * 2 + which) * c.kv_heads + head) << c.page_shift) + slot) * (D / 2);
}
ATB_DEVICE __nv_bfloat16* scales_at(const Cache& c, int page, int head, int slot) {
  return c.scales + ((((long long)page * c.kv_heads + head) << c.page_shift) + slot) * 4;
}

// 8 elements as they lie in memory
template <typename T>
struct Piece {
  uint4 u[sizeof(T) / 2];
  ATB_DEVICE void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  ATB_DEVICE void get(float (&x)[8]) const {
    const T* h = reinterpret_cast<const T*>(u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(h[i]);
  }
};
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

constexpr int SMALL = 128;      // threads of a block of the two kernels below: a few heads of one token

// A head of a token is D / 16 lanes: each has 8 dims of the first half and the 8 of the second half that they turn with.
// The result is that of separately rounded fp32 operations (no fused multiply-add, true division), so that the codes are those of
// the formula evaluated operation by operation, and do not depend on how a compiler contracts it. The scale is rounded to bf16
// before the codes are taken: the code is the nearest one of the scale that is kept. Bound by memory where there are many tokens:
// so a division is a product with the reciprocal, and only a quotient that comes within 1e-5 of the middle of two codes (the
// product is off by 2e-6 at most) is divided (a true division for each took 78 us for 10900 tokens of 48 heads, 53 us
// now: 4.4 TB/s).
template <typename T, int D, int PER>
__global__ void __launch_bounds__(SMALL, PER == 1 || sizeof(T) == 4 ? 1 : 7) kv4_append_kernel(const T* qkv, T* q_out, Cache c, const int* seq, const int* pos,
                                                           const float* cosT, const float* sinT, int positions, int n_q,
                                                           long long token_stride, int* status) {
  grid_go();
  grid_wait();
  constexpr int L = D / 16, HALF = D / 2, EACH = SMALL / L;
  const int heads = n_q + 2 * c.kv_heads, l = threadIdx.x % L, h0 = blockIdx.y * (EACH * PER) + threadIdx.x / L;
  const long long t = blockIdx.x;
  const int before = *status, row = seq ? seq[t] : (int)t;
  int p = pos[t], page = -1;
  Piece<T> x[PER][2];              // 8 dims of the first half of head h0 + j EACH, 8 of the second
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (h0 + j * EACH < heads) {
      const T* src = qkv + t * token_stride + (long long)(h0 + j * EACH) * D + l * 8;
      x[j][0].load(src);
      x[j][1].load(src + HALF);
    }
  if (p >= 0) {
    page = page_of(c, row, p);
    if (page < 0 || (cosT && p >= positions)) {
      atomicCAS(status, 0, (int)ATB_ERR_BAD_INDEX);
      page = -1;
      p = -1;
    }
  }
  float cs[8], sn[8];
  const bool turn = cosT && p >= 0 && h0 < n_q + c.kv_heads;
  if (turn) {
    load8<float>(cosT + (long long)p * HALF + l * 8, cs);
    load8<float>(sinT + (long long)p * HALF + l * 8, sn);
  }
  const bool failed = warp_uniform(before) != 0;       // one answer for the lanes of a head; every lane has to ask
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int h = h0 + j * EACH;
    const bool live = h < heads && !failed;
    float a[8], b[8];
    x[j][0].get(a);
    x[j][1].get(b);
    if (turn && h < n_q + c.kv_heads) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = a[i], v = b[i];
        a[i] = __fsub_rn(__fmul_rn(u, cs[i]), __fmul_rn(v, sn[i]));
        b[i] = __fadd_rn(__fmul_rn(v, cs[i]), __fmul_rn(u, sn[i]));
      }
    }
    if (live && h < n_q) {
      T* dst = q_out + (t * n_q + h) * D + l * 8;
      store8<T>(dst, a);
      store8<T>(dst + HALF, b);
    }
    const bool kept = live && h >= n_q && page >= 0;
    if (!__any_sync(0xffffffffu, kept)) continue;
    float lo = 0.f, hi = 0.f;
    if (kept) {
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
    if (kept) {
      const __nv_bfloat16 scale = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f)), low = __float2bfloat16_rn(lo);
      const float s = __bfloat162float(scale), m = __bfloat162float(low);
      uint32_t w[2] = {0u, 0u};
      if (s > 0.f) {
        const float inv = __frcp_rn(s), round = 12582912.f;       // 1.5 * 2^23: adding it leaves the nearest integer, ties to even
        float off = s < 1e-30f ? 1.f : 0.f;                       // (a reciprocal that is not exact enough, or infinite)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float d = __fsub_rn(i < 8 ? a[i] : b[i - 8], m);
          const float y = fminf(fmaxf(__fmul_rn(d, inv), 0.f), 15.f);
          const float r = __fadd_rn(y, round);
          off = fmaxf(off, fabsf(__fsub_rn(y, __fsub_rn(r, round))));
          w[i / 8] |= (__float_as_uint(r) & 15u) << (4 * (i % 8));
        }
        if (off > 0.49999f) {
          w[0] = w[1] = 0u;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float d = __fsub_rn(i < 8 ? a[i] : b[i - 8], m);
            w[i / 8] |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(d, s)), 0.f), 15.f) << (4 * (i % 8));
          }
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
  }
}

// What the cache stands for at given tokens: a lane turns 8 codes of the keys and of the values of PER tokens into two 16-byte
// pieces each. Positions, pages and codes follow one another, so the tokens' are asked for side by side.
template <typename T, int D, int PER>
__global__ void __launch_bounds__(SMALL) kv4_read_kernel(T* k, T* v, Cache c, const int* seq, const int* pos, int tokens,
                                                         int* status) {
  grid_go();
  grid_wait();
  constexpr int L = D / 8;
  const int l = threadIdx.x % L, h = blockIdx.y * (SMALL / L) + threadIdx.x / L, t0 = blockIdx.x * PER;
  const int before = *status;
  int p[PER], page[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) p[j] = t0 + j < tokens ? pos[t0 + j] : -1;
#pragma unroll
  for (int j = 0; j < PER; ++j) page[j] = p[j] >= 0 ? page_of(c, seq ? seq[t0 + j] : t0 + j, p[j]) : -1;
  if (h >= c.kv_heads || before != 0) return;
  uint2 sc[PER];
  uint32_t w[PER][2];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    sc[j] = make_uint2(0u, 0u);
    w[j][0] = w[j][1] = 0u;
    if (page[j] >= 0) {
      const int slot = p[j] & ((1 << c.page_shift) - 1);
      sc[j] = *reinterpret_cast<const uint2*>(scales_at(c, page[j], h, slot));
#pragma unroll
      for (int i = 0; i < 2; ++i) w[j][i] = *reinterpret_cast<const uint32_t*>(codes_at<D>(c, page[j], i, h, slot) + l * 4);
    } else if (p[j] >= 0) {
      atomicCAS(status, 0, (int)ATB_ERR_BAD_INDEX);
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (t0 + j >= tokens) break;
    const long long at = ((long long)(t0 + j) * c.kv_heads + h) * D + l * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = unpack_bf16x2(i ? sc[j].y : sc[j].x);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)((w[j][i] >> (4 * e)) & 15u) * f.x + f.y;
      store8<T>((i ? v : k) + at, x);
    }
  }
}

// ----------------------------------------------------------------------------------
// Attention
// ----------------------------------------------------------------------------------
// Query i of sequence b's S newest tokens sees its keys j < lengths[b] - S + i + 1. The g query heads of a key/value head times
// the S tokens are the columns of one matrix product: n = i g + h, in tiles of 8 or 16.
//
// The work is one row of units: the tiles of 32 tokens of a sequence, once per head and column tile, one sequence behind another.
// Every block takes an equal run of it, which it finds for itself from the lengths on the device (they need not be known on the
// host), so that long and short sequences fill the GPU alike. A run is cut into segments where a sequence (of a head) ends;
// what a segment costs beside its tiles counts as START units before the first (5, 8 and 12 of them: 32 sequences of up to 4096
// tokens 32.0, 30.3 and 30.3 us, two of 100k 60.3, 58.6 and 58.6). A segment that is a whole sequence is finished
// in place; of the others, the run's first and last, a block leaves sums, maximum and denominator, which a second kernel joins in
// the order of the blocks.
constexpr int WARPS = 4, TILE = 32, START = 12;
constexpr float SLACK = 4.f;       // powers of two by which a score may exceed the maximum that is kept
constexpr int LEAST_E = 24, AHEAD_E = 12;      // exponent fields of value scales: the least, and how far one may lie above what its weight leaves

using Cut = Runs<TILE, START, WARPS>;

// 16-byte pieces from global to shared memory by the copy unit (both addresses and the size multiples of 16)
ATB_DEVICE void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
ATB_DEVICE void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero.
ATB_DEVICE void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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
  if constexpr (WORDS == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    r.w[0] = u.x; r.w[1] = u.y; r.w[2] = u.z; r.w[3] = u.w;
  }
  return r;
}

struct AttnArgs {
  Cache c;
  const int* lengths;
  const void* q;
  void* out;
  float* lse;                 // [rows][heads][S] or nullptr
  float* partial;             // sums [2 ctas][columns of a tile][D], then maximum and denominator [2 ctas][columns][2]
  int2* owners;               // first and last block of each [row][head and column tile]
  long long q_batch, q_token; // strides of q, elements
  int S, heads, group;
  float scale_log2;           // softmax scale * log2(e)
  int ctas;                   // blocks that the work is cut for; 0: a block takes whole sequences (of a head), one after another
  int* status;
};

// Both products run on the warp's matrix instruction (16 x 8 x 16, fp16, fp32 sums) with the codes as its 16-row operand. A
// code needs no conversion: its 4 bits, alone in the low bits of a half, are the fp16 number code * 2^-24, and four places
// further up code * 2^-20; so eight codes cost four ANDs and a shift. The other operand takes the powers of two and everything
// else that a value has:
//   s[t, n] = ks[t] (q[n] . code[t]) + km[t] sum(q[n])
//   o[d, n] = sum_t (p[t, n] vs[t]) (code[t, d] - 8) + sum_t p[t, n] (vm[t] + 8 vs[t])
// q is scaled by a power of two to at most 2^15 before it is rounded to fp16 (bf16 and fp16 values stay exact down to 2^-29 of
// the largest, and in range below 2^117), p vs by a power of two that runs with the softmax, for each column its own: by the largest
// exponent of a value's scale so far, as long as that is not 2^12 above the largest p vs (a token without weight, however large its
// values, takes no bits from the others; nor does one that a column does not see). 11 bits of p vs are kept, and absolutely
// 2^-20 of the largest at least. The 8s are taken off as products of the same rounded numbers (a row of 8s in the place of codes), so that
// their rounding errors weigh as much as a value and not as a code: fp16 results of 5 tokens, 64-wide heads, were off by 3.6e-4
// without it, 2.3e-4 now, of which rounding to fp16 takes 2.1e-4. Sums, maxima and denominators are fp32.
//
// A warp has every fourth tile of a segment. Its tiles come through a ring of its own in shared memory, filled by the copy unit
// STAGES tiles ahead. Beside the copies the integer pipe has most to do: 5 operations for 8 codes of a key, 6 of a value.
// So the rest of a tile is kept short: scores are taken relative to the running maximum, which is looked at by one vote, and only
// the tiles at a sequence's end are masked. The maximum that is kept may be exceeded by 2^4 before everything is rescaled: a warp
// sees few enough tiles for a new maximum in half of them. Row i of 16 tokens' products is token order(i): a lane then reads its
// values' words without a bank conflict worse than two ways.
// Measured, 32 query heads on 8 of 128: two sequences of 100k tokens (207 MB) 58.6 us, 3.5 TB/s; 32 of up to 4096 (64 MB) 30.3 us. With
// the arithmetic left out, the copies, waits and starts take 50 and 23 us, and a library's sum over as many bytes 41 and 20: memory
// bounds the kernel, and of the arithmetic (an instruction every other clock, the integer pipe busy 57 % of the time) what a block
// does while it has no copies on their way. Loading tiles into registers a warp's tile at a time took 99 and 51 us; a third stage,
// queries in shared memory, a fifth block an SM, or the products of the next tile beside the sums of this one were no faster.
template <int D, int NT>
struct Shape {
  static constexpr int COLS = 8 * NT, STAGE = TILE * D + TILE * 8, STAGES = NT == 1 ? 2 : 4, RING = WARPS * STAGES * STAGE;
  static constexpr int BLOCKS = NT == 1 ? 4 : 2;       // of an SM: 128 or 255 registers
};
ATB_DEVICE int order(int i) {
  const int k = (i & 7) >> 1;
  return (i & 8) + ((i & 1) ? (k ^ 1) + 4 : k);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(WARPS * 32, Shape<D, NT>::BLOCKS) kv4_attention_kernel(AttnArgs a) {
  using Sh = Shape<D, NT>;
  constexpr int KW = D / 32, VW = D / 64, COLS = Sh::COLS, MT = D / 16, STAGES = Sh::STAGES;
  static_assert(WARPS * COLS * (D + 4) * 4 <= Sh::RING, "the warps' sums lie in the place of the ring");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sh_m[WARPS][COLS], sh_l[WARPS][COLS];
  __shared__ uint64_t bars[WARPS][STAGES];
  __shared__ int abort_flag;
  const Cache& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, q4 = lane & 3;
  uint8_t* const ring = smem + warp * (STAGES * Sh::STAGE);
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane < STAGES) mbar_init(&bars[warp][lane], 1);
  mbar_fence_init();
  grid_go();
  grid_wait();
  const int failed = threadIdx.x == 0 ? *a.status : 0;       // on its way beside the lengths
  const int columns = a.S * a.group, col_tiles = (columns + COLS - 1) / COLS, per = col_tiles * c.kv_heads;
  Plan plan{};
  long long u = blockIdx.x, run_end = (long long)c.rows * per;       // whole sequences: their numbers
  if (a.ctas > 0) {
    plan = Cut::plan(c, a.lengths, per, a.ctas, a.status);
    u = plan.begin(blockIdx.x);
    run_end = plan.begin(blockIdx.x + 1);
  }
  if (__syncthreads_or(failed != 0)) return;       // one answer for the block: others may fail meanwhile
  if (a.ctas > 0 && (int)blockIdx.x >= plan.ctas) return;
  uint32_t loads = 0;            // tiles that this warp has taken from its ring

  // A tile is two pieces of 16 tokens, each in one page, of three copies: keys, values, scales. Lane 3 p + x has copy x of piece p.
  // Where a page holds a whole tile, the first piece's copies bring both (two sequences of 100k tokens: 60.3 us without, 58.6).
  const int piece = lane / 3, what = lane - 3 * piece;
  const bool copies = lane < 6;
  const long long page_stride = ((what < 2 ? (long long)c.kv_heads * D : c.kv_heads * 8LL) << c.page_shift);
  const bool whole_tiles = (1 << c.page_shift) >= TILE;
  const int token_bytes = what < 2 ? D / 2 : 8;
  const int dst_at = (what < 2 ? what * (TILE * D / 2) : TILE * D) + piece * 16 * token_bytes;

  while (u < run_end) {
    int b, len, hc, tiles, t_first = 0, t_last;       // the segment: tiles [t_first, t_last) of a sequence
    long long begin = 0;
    if (a.ctas > 0) {
      long long first;
      Cut::find(c, a.lengths, per, u, b, len, first, a.status);
      tiles = Cut::tiles_of(len);
      hc = (int)((u - first) / (START + tiles));
      begin = first + (long long)hc * (START + tiles);
      t_first = max(0, (int)(u - begin) - START);
      t_last = (int)min(run_end - begin - START, (long long)tiles);
      u = begin + START + t_last;
      if (t_last <= t_first) break;      // the run ends before the first tile
    } else {
      b = (int)(u / per);
      hc = (int)(u - (long long)b * per);
      len = seen_length(c, a.lengths, b, a.status);
      t_last = tiles = Cut::tiles_of(len);
      u += gridDim.x;
    }
    const int head = hc % c.kv_heads, col_tile = hc / c.kv_heads;
    const bool whole = t_first == 0 && t_last == tiles;
    if (a.ctas > 0 && t_first == 0 && threadIdx.x == 0)
      a.owners[(long long)b * per + hc] = make_int2(blockIdx.x, plan.owner(begin + START + tiles - 1));
    const int mine = len == 0 ? 0 : max(0, (t_last - t_first - warp + WARPS - 1) / WARPS);
    const int* const row = c.table + b * c.table_stride;
    const uint8_t* const src_at = what < 2 ? codes_at<D>(c, 0, what, head, 0) : reinterpret_cast<uint8_t*>(scales_at(c, 0, head, 0));

    // pages of the warp's pieces 2 j to 2 j + 31: two of each tile
    auto pages_from = [&](int j) {
      const int t = (t_first + warp + (j + (lane >> 1)) * WARPS) * TILE + (lane & 1) * 16;
      int page = 0;
      if (j + (lane >> 1) < mine && t < len) {
        page = row[t >> c.page_shift];
        if (page < 0 || page >= c.pages) {
          atomicCAS(a.status, 0, (int)ATB_ERR_BAD_INDEX);
          page = 0;
        }
      }
      return page;
    };
    int pages = pages_from(0);
    auto fetch = [&](int j) {      // by the whole warp: tile j into the ring
      if (j >= mine) return;
      if (j > 0 && (j & 15) == 0) pages = pages_from(j);
      const int page = __shfl_sync(0xffffffffu, pages, (2 * j + piece) & 31);
      const int t = (t_first + warp + j * WARPS) * TILE + piece * 16;
      const uint32_t s = (loads + j) % STAGES;
      const bool both = t - piece * 16 + 16 < len;         // the second piece may lie behind the sequence, and have no page
      if (lane == 0) mbar_expect_tx(&bars[warp][s], both ? Sh::STAGE : Sh::STAGE / 2);
      __syncwarp();
      const int tokens = both && whole_tiles ? TILE : 16;
      if (copies && t < len && (tokens == 16 || piece == 0))
        bulk_load(ring + s * Sh::STAGE + dst_at, src_at + page * page_stride + (t & ((1 << c.page_shift) - 1)) * token_bytes,
                  tokens * token_bytes, &bars[warp][s]);
    };
    for (int j = 0; j < STAGES; ++j) fetch(j);

    // queries: column 8 j + r, this lane's quarter of the dims; odd places of a word carry 2^-4
    uint32_t qf[NT][KW][4];
    float cs[NT][2], bs[NT][2];      // factors of the products and sum(q) of the columns 8 j + 2 q4 + {0, 1}
    int limit[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = col_tile * COLS + 8 * j + r;
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
      const int e = top > 0.f ? min(max((__float_as_int(top) >> 23) - 127, -100), 116) : 0;   // top < 2^(e + 1)
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
        const int col = col_tile * COLS + 8 * j + 2 * q4 + o;
        limit[j][o] = min(len, len - a.S + col / a.group + 1);
      }
    }
    const int all_see = len - a.S + col_tile * COLS / a.group + 1;      // tokens that every column of the tile sees

    // running maximum of the scores (m), sums of p, of p times the values' minima and of p times their scaled codes; `ref` is what
    // scores are taken relative to: m, or 0 where there is none yet
    float o_acc[NT][MT][4], eights[NT][4], m[NT][2], ref[NT][2], l[NT][2], z[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o_acc[j][i][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) eights[j][e] = 0.f;
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        m[j][o] = -INFINITY;
        ref[j][o] = l[j][o] = z[j][o] = 0.f;
      }
    }
    int top_e[NT][2], least_e = LEAST_E;       // exponent fields that p vs is scaled by, and the lane's least one
#pragma unroll
    for (int j = 0; j < NT; ++j) top_e[j][0] = top_e[j][1] = LEAST_E;
    bool unset = true;     // whether a column has no maximum yet

    auto tile = [&](const uint8_t* src, int t0, auto masked) {
      constexpr bool MASK = decltype(masked)::value;
      float s[2][NT][4];
      float2 vs[4];
      float over = 0.f;
      uint32_t most_scale = 0;       // bf16 bits
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const Words<KW> x = load_words<KW>(src + (16 * p + order(r)) * (D / 2) + q4 * (KW * 4));
        const Words<KW> y = load_words<KW>(src + (16 * p + order(r) + 8) * (D / 2) + q4 * (KW * 4));
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          const uint32_t xs = x.w[k] >> 8, ys = y.w[k] >> 8;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (k == 0)
              mma_f16_first(s[p][n], x.w[k] & 0x000F000Fu, y.w[k] & 0x000F000Fu, x.w[k] & 0x00F000F0u, y.w[k] & 0x00F000F0u,
                            qf[n][k][0], qf[n][k][1]);
            else
              mma_f16(s[p][n], x.w[k] & 0x000F000Fu, y.w[k] & 0x000F000Fu, x.w[k] & 0x00F000F0u, y.w[k] & 0x00F000F0u,
                      qf[n][k][0], qf[n][k][1]);
            mma_f16(s[p][n], xs & 0x000F000Fu, ys & 0x000F000Fu, xs & 0x00F000F0u, ys & 0x00F000F0u, qf[n][k][2], qf[n][k][3]);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = 16 * p + order(r) + 8 * i;
          uint2 sc = *reinterpret_cast<const uint2*>(src + TILE * D + t * 8);
          if (MASK && t0 + t >= len) sc = make_uint2(0u, 0u);           // places behind the last token hold anything
          const float2 ks = unpack_bf16x2(sc.x);
          vs[2 * p + i] = unpack_bf16x2(sc.y);
          most_scale = max(most_scale, sc.y & 0x7fffu);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              float& v = s[p][n][2 * i + o];
              v = fmaf(ks.x * cs[n][o], v, fmaf(ks.y, bs[n][o], -ref[n][o]));
              if (MASK && t0 + t >= limit[n][o]) v = -INFINITY;
              over = fmaxf(over, v);
            }
        }
      }
      if (__any_sync(0xffffffffu, over > SLACK || (int)(most_scale >> 7) > least_e || unset)) {
        uint32_t range = 0;            // the largest exponent, and 255 less the least of those that are not 0
        int e_vs[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = (__float_as_int(vs[i].x) >> 23) & 255;
          e_vs[i] = e == 255 ? 0 : e;       // an infinity is not for the queries that do not see it
          range = __vmaxu2(range, e_vs[i] > 0 ? e_vs[i] | (255 - e_vs[i]) << 16 : 0);
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) range = __vmaxu2(range, __shfl_xor_sync(0xffffffffu, range, o));
        const int e_most = range & 0xffff, e_min = 255 - (int)(range >> 16);
        bool apart = false;            // whether exponents of a column lie so far apart that the weights have to be looked at
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int o = 0; o < 2; ++o)
            apart = apart || max(top_e[n][o], e_most) - (m[n][o] == -INFINITY ? e_min : min(top_e[n][o], e_min)) > AHEAD_E;
        apart = __any_sync(0xffffffffu, apart);
        least_e = 255;
        unset = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float f[2];
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            float most = -INFINITY;
#pragma unroll
            for (int p = 0; p < 2; ++p) most = fmaxf(most, fmaxf(s[p][n][o], s[p][n][2 + o]));
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, k));
            const float to = fmaxf(m[n][o], ref[n][o] + most), by = (to == -INFINITY ? 0.f : to) - ref[n][o];
            const bool first = m[n][o] == -INFINITY;
            f[o] = first ? 0.f : fast_exp2(-by);
            m[n][o] = to;
            ref[n][o] += by;
            unset = unset || to == -INFINITY;
            l[n][o] *= f[o];
            z[n][o] *= f[o];
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i >> 1][n][2 * (i & 1) + o] -= by;
            int e = max(top_e[n][o], e_most);
            if (apart) {
              int weighed = first ? -1000 : top_e[n][o] - __float2int_rd(by);       // p vs so far is below 2^(this - 126)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float v = s[i >> 1][n][2 * (i & 1) + o];
                if (v > -INFINITY) weighed = max(weighed, e_vs[i] + __float2int_ru(fmaxf(v, -300.f)));
              }
#pragma unroll
              for (int k = 4; k < 32; k <<= 1) weighed = max(weighed, __shfl_xor_sync(0xffffffffu, weighed, k));
              e = max(LEAST_E, min(e, weighed + AHEAD_E));
            }
            f[o] *= __int_as_float((127 + max(min(top_e[n][o] - e, 126), -126)) << 23);
            top_e[n][o] = e;
            least_e = min(least_e, e);
          }
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o_acc[n][i][e] *= f[e & 1];
#pragma unroll
          for (int e = 0; e < 4; ++e) eights[n][e] *= f[e & 1];
        }
      }
      float up[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int o = 0; o < 2; ++o) up[n][o] = pow2(137 + 4 - (int)SLACK - top_e[n][o]);      // 2^(15 - SLACK) / 2^(exponent + 1)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint32_t pf[NT][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = 16 * p + order(r) + 8 * i;
          const float scale = vs[2 * p + i].x, middle = fmaf(8.f, vs[2 * p + i].x, vs[2 * p + i].y);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float pv[2];
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const float w = fast_exp2(s[p][n][2 * i + o]);
              const bool seen = !MASK || t0 + t < limit[n][o];
              l[n][o] += w;
              z[n][o] = seen ? fmaf(w, middle, z[n][o]) : z[n][o];
              pv[o] = seen ? w * scale * up[n][o] : 0.f;      // (w scale is in range, scale up need not be)
            }
            pf[n][i] = transpose_8x8(pack_f16x2(pv[0], pv[1]));
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
          mma_f16(eights[n], 0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u, pf[n][0], pf[n][1]);
        Words<VW> vc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          vc[i] = load_words<VW>(src + TILE * D / 2 + (16 * p + order(2 * q4 + (i & 1) + 8 * (i >> 1))) * (D / 2) + r * (VW * 4));
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          // words of two tokens side by side: places 0 to 3 of both, then 4 to 7
          const uint32_t lo0 = __byte_perm(vc[0].w[k], vc[1].w[k], 0x5410), hi0 = __byte_perm(vc[0].w[k], vc[1].w[k], 0x7632);
          const uint32_t lo1 = __byte_perm(vc[2].w[k], vc[3].w[k], 0x5410), hi1 = __byte_perm(vc[2].w[k], vc[3].w[k], 0x7632);
          const uint32_t x[4] = {lo0, lo0 >> 8, hi0, hi0 >> 8}, y[4] = {lo1, lo1 >> 8, hi1, hi1 >> 8};
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma_f16(o_acc[n][4 * k + i], x[i] & 0x000F000Fu, x[i] & 0x00F000F0u, y[i] & 0x000F000Fu, y[i] & 0x00F000F0u,
                      pf[n][0], pf[n][1]);
        }
      }
    };

    bool arrived = true;
    for (int j = 0; j < mine; ++j) {
      const uint32_t stage = (loads + j) % STAGES, phase = ((loads + j) / STAGES) & 1;
      const int t0 = (t_first + warp + j * WARPS) * TILE;
      arrived = mbar_wait_warp(&bars[warp][stage], phase, &abort_flag, a.status);
      if (!arrived) break;
      if (t0 + TILE <= all_see) tile(ring + stage * Sh::STAGE, t0, std::false_type());
      else tile(ring + stage * Sh::STAGE, t0, std::true_type());
      __syncwarp();
      fetch(j + STAGES);
    }
    loads += mine;

    // the warps' sums, in their order, in the place of the rings: every copy has arrived and been read
    float (*const sh_o)[COLS][D + 4] = reinterpret_cast<float (*)[COLS][D + 4]>(smem);
    if (__syncthreads_or(!arrived)) {
      // a copy did not come in time: nothing more is asked for or stored, and those on their way may land before the block ends
      const uint64_t t_start = globaltimer_ns();
      while (globaltimer_ns() - t_start < 200000ull) __nanosleep(1000);
      return;
    }
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
        // what p vs was scaled by, taken back; codes stand at 2^-24, the odd places at 2^-20 (two factors: neither overflows alone)
        const float f = pow2(top_e[j][o] - 137 - 4 + (int)SLACK);
#pragma unroll
        for (int i = 0; i < MT; ++i)
          *reinterpret_cast<float2*>(&sh_o[warp][col][r * (D / 8) + 2 * i]) =
              make_float2(fmaf((o_acc[j][i][o] - eights[j][o]) * 16777216.f, f, z[j][o]),
                          fmaf(fmaf(-16.f, eights[j][o], o_acc[j][i][2 + o]) * 1048576.f, f, z[j][o]));
      }
    }
    __syncthreads();
    const long long slot = 2LL * blockIdx.x + (t_first == 0);        // a sequence that goes on, or one that begins, in this block
    for (int x = threadIdx.x; x < COLS * (D / 4); x += WARPS * 32) {
      const int col = x / (D / 4), d = (x - col * (D / 4)) * 4, n = col_tile * COLS + col;
      if (n >= columns) continue;
      float top = sh_m[0][col];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) top = fmaxf(top, sh_m[k][col]);
      float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float f = sh_m[k][col] == -INFINITY ? (sh_l[k][col] == 0.f ? 0.f : 1.f) : fast_exp2(sh_m[k][col] - top);
        const float4 v = *reinterpret_cast<const float4*>(&sh_o[k][col][d]);
        sum += f * sh_l[k][col];
        o[0] += f * v.x;
        o[1] += f * v.y;
        o[2] += f * v.z;
        o[3] += f * v.w;
      }
      if (!whole) {
        *reinterpret_cast<float4*>(a.partial + (slot * COLS + col) * D + d) = make_float4(o[0], o[1], o[2], o[3]);
        if (d == 0)
          *reinterpret_cast<float2*>(a.partial + 2LL * a.ctas * COLS * D + (slot * COLS + col) * 2) = make_float2(top, sum);
      } else {
        const int i = n / a.group, h = head * a.group + n - i * a.group;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(o[e] * inv);
        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + (((long long)b * a.S + i) * a.heads + h) * D + d) =
            *reinterpret_cast<const uint2*>(y);
        if (d == 0 && a.lse) a.lse[((long long)b * a.heads + h) * a.S + i] = (top + log2f(sum)) * 0.69314718056f;
      }
    }
    if (u < run_end) {
      fence_proxy_async_smem();      // the sums were written by the threads, the next tiles come by the copy unit
      __syncthreads();
    }
  }
}

// Sequences (of a head and a column tile: a block) that several blocks worked on. Bound by latency: the blocks' results are read
// eight at a time, independent of one another.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(256) kv4_join_kernel(AttnArgs a, int per) {
  constexpr int COLS = 8 * NT, EACH = 8;
  grid_go();
  grid_wait();
  const int2 own = a.owners[blockIdx.x];
  const bool failed = *a.status != 0;
  // (behind a kernel that left early there may be anything)
  if (__syncthreads_or(failed) || own.x < 0 || own.y >= a.ctas || own.x >= own.y) return;
  const int columns = a.S * a.group, b = blockIdx.x / per, hc = blockIdx.x - b * per;
  const int head = hc % a.c.kv_heads, col_tile = hc / a.c.kv_heads;
  const float* const stats = a.partial + 2LL * a.ctas * COLS * D;
  for (int x = threadIdx.x; x < COLS * (D / 4); x += 256) {
    const int col = x / (D / 4), d = (x - col * (D / 4)) * 4, n = col_tile * COLS + col;
    if (n >= columns) continue;
    float top = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = own.x; k0 <= own.y; k0 += EACH) {
      float2 ml[EACH];
      float4 v[EACH];
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        const int at = (2 * min(k0 + k, own.y) + (k0 + k == own.x)) * COLS + col;
        ml[k] = *reinterpret_cast<const float2*>(stats + 2LL * at);
        v[k] = *reinterpret_cast<const float4*>(a.partial + (long long)at * D + d);
        if (k0 + k > own.y) ml[k] = make_float2(-INFINITY, 0.f);
      }
      float to = top;
#pragma unroll
      for (int k = 0; k < EACH; ++k) to = fmaxf(to, ml[k].x);
      const float down = top == -INFINITY ? (sum == 0.f ? 0.f : 1.f) : fast_exp2(top - to);
      sum *= down;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= down;
      top = to;
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        if (k0 + k > own.y) continue;
        const float f = ml[k].x == -INFINITY ? (ml[k].y == 0.f ? 0.f : 1.f) : fast_exp2(ml[k].x - top);
        sum += f * ml[k].y;
        o[0] += f * v[k].x;
        o[1] += f * v[k].y;
        o[2] += f * v[k].z;
        o[3] += f * v[k].w;
      }
    }
    const int i = n / a.group, h = head * a.group + n - i * a.group;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(o[e] * inv);
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + (((long long)b * a.S + i) * a.heads + h) * D + d) =
        *reinterpret_cast<const uint2*>(y);
    if (d == 0 && a.lse) a.lse[((long long)b * a.heads + h) * a.S + i] = (top + log2f(sum)) * 0.69314718056f;
  }
}

Cache cache_of(void* codes, void* scales, const void* table, long long table_stride, int rows, int width, int pages,
               int kv_heads, int page_shift) {
  return Cache{{(const int*)table, table_stride, rows, width, pages, kv_heads, page_shift}, (uint8_t*)codes, (__nv_bfloat16*)scales};
}

template <typename T, int D>
int launch_append(const void* qkv, void* q, const Cache& c, const void* seq, const void* pos, const void* cosT, const void* sinT,
                  int positions, int tokens, int n_q, long long stride, cudaStream_t st, int* status) {
  const int each = SMALL / (D / 16), heads = n_q + 2 * c.kv_heads;
  // where there are more blocks than the GPU holds, a thread has three heads: more loads on their way, one look at the page table
  // and the angles (one head each: 82 us for 10900 tokens of 48 heads and their reading back, three: 70)
  const bool many = (long long)tokens * ((heads + each - 1) / each) > 148 * 16 && heads > each;
  const int blocks = many ? (heads + 3 * each - 1) / (3 * each) : (heads + each - 1) / each;
  if (blocks > 65535) return -2;
  return launched(launch_after(many ? kv4_append_kernel<T, D, 3> : kv4_append_kernel<T, D, 1>, dim3(tokens, blocks), SMALL, 0, st, 1,
                      (const T*)qkv, (T*)q, c, (const int*)seq, (const int*)pos, (const float*)cosT, (const float*)sinT, positions,
                      n_q, stride, status));
}
template <typename T, int D>
int launch_read(void* k, void* v, const Cache& c, const void* seq, const void* pos, int tokens, cudaStream_t st, int* status) {
  const int each = SMALL / (D / 8), blocks = (c.kv_heads + each - 1) / each;
  if (blocks > 65535) return -2;
  const bool many = (long long)tokens * blocks > 148 * 16 * 2;
  return launched(launch_after(many ? kv4_read_kernel<T, D, 4> : kv4_read_kernel<T, D, 1>, dim3(many ? (tokens + 3) / 4 : tokens, blocks), SMALL,
                      0, st, 1, (T*)k, (T*)v, c, (const int*)seq, (const int*)pos, tokens, status));
}

template <typename T, int D, int NT>
int launch_attention(AttnArgs a, cudaStream_t st) {
  using Sh = Shape<D, NT>;
  static std::atomic<unsigned long long> allowed{0};       // devices on which the kernel may have its shared memory
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return launched(cudaErrorInvalidDevice);
  const unsigned long long bit = 1ull << (device & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    const int rc = launched(cudaFuncSetAttribute(kv4_attention_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::RING));
    if (rc != 0) return rc;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  const long long per = (a.S * a.group + Sh::COLS - 1) / Sh::COLS * (long long)a.c.kv_heads;
  const long long room = (((long long)a.c.width << a.c.page_shift) + TILE - 1) / TILE;       // tiles that a sequence can have
  const long long most = (START + (room > 1 ? room : 1)) * a.c.rows * per, runs = a.c.rows * per;
  if (runs > 0x7fffffffLL) return -2;
  // sequences of up to 256 tokens are not cut: two tiles a warp take less than a join and what the cutting needs to know
  const bool cut = room > 8;
  if (cut && !a.partial) return -1;
  a.ctas = 148 * Sh::BLOCKS;
  if (cut) a.owners = reinterpret_cast<int2*>(a.partial + 2LL * a.ctas * Sh::COLS * (D + 2));
  const unsigned grid = (unsigned)(most < a.ctas ? most : a.ctas);
  if (!cut) a.ctas = 0;
  const int rc = launched(launch_after(kv4_attention_kernel<T, D, NT>, dim3(cut || runs > grid ? grid : (unsigned)runs), WARPS * 32,
                                       Sh::RING, st, 1, a));
  if (rc != 0 || !cut) return rc;
  return launched(launch_after(kv4_join_kernel<T, D, NT>, dim3((unsigned)runs), 256, 0, st, 1, a, (int)per));
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

// Floats of the workspace of atb_kv4_attention: two segments a block, and two numbers a sequence.
extern "C" long long atb_kv4_attention_scratch(int rows, int heads, int kv_heads, int S, int head_dim) {
  const int columns = S * (heads / kv_heads), cols = columns > 8 ? 16 : 8, blocks = columns > 8 ? Shape<128, 2>::BLOCKS : Shape<128, 1>::BLOCKS;
  return 2LL * 148 * blocks * cols * (head_dim + 2) + 2LL * rows * kv_heads * ((columns + cols - 1) / cols);
}

extern "C" int atb_kv4_attention(const void* q, void* out, void* lse, void* codes, void* scales, const void* table,
                                 const void* lengths, void* partial, int S, int heads, int kv_heads, int head_dim,
                                 int page_shift, int pages, int rows, int width, long long table_stride,
                                 long long q_batch, long long q_token, float scale, int dtype, void* stream, void* status) {
  if (rows <= 0 || S <= 0) return 0;
  AttnArgs a;
  a.c = cache_of(codes, scales, table, table_stride, rows, width, pages, kv_heads, page_shift);
  a.lengths = (const int*)lengths;
  a.q = q;
  a.out = out;
  a.owners = nullptr;
  a.lse = (float*)lse;
  a.partial = (float*)partial;
  a.q_batch = q_batch;
  a.q_token = q_token;
  a.S = S;
  a.heads = heads;
  a.group = heads / kv_heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = (int*)status;
  const bool two = S * a.group > 8;
#define ATTN(T, D) \
  return two ? launch_attention<T, D, 2>(a, (cudaStream_t)stream) : launch_attention<T, D, 1>(a, (cudaStream_t)stream)
  if (dtype == 0 && head_dim == 64) ATTN(__nv_bfloat16, 64);
  if (dtype == 0 && head_dim == 128) ATTN(__nv_bfloat16, 128);
  if (dtype == 1 && head_dim == 64) ATTN(__half, 64);
  if (dtype == 1 && head_dim == 128) ATTN(__half, 128);
#undef ATTN
  return -1;
}
