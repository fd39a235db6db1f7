// Paged key/value cache in 16 bits: append with rotation, attention of the newest tokens, eviction of tokens with little weight.
//
// One layer's cache is T [pages][2][kv heads][page size][D]: 0: keys, 1: values.
#include <atomic>
#include <cooperative_groups.h>
#include <type_traits>
#include "paged.cuh"

namespace {
using namespace atb;
namespace cg = cooperative_groups;

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
// contracts it. Bound by memory where there are many tokens (12321 of 48 heads: 52.9 us, 6.2 TB/s; one head a thread 56.4), by latency for
// the one token of a step (64 sequences: 1.9 us on the device).
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
// Query i of sequence b's S newest tokens sees its keys j < lengths[b] - S + i + 1. The g query heads of a key/value head times
// the S tokens are the columns of one matrix product: n = i g + h, in tiles of 8, 16 or 32.
//
// The work is cut into equal runs over the GPU (paged.cuh). A segment that is a whole sequence (of a head and column tile) is
// finished in place; of the others, a run's first and last, a block leaves sums, maximum and denominator, which a second kernel joins
// in the order of the blocks. (START of 6, 12, 24 and 40 tiles: 32 sequences of up to 4096 59.0, 45.7, 44.8 and 46.2 us, one of 1531 10.0,
// 9.9, 9.2 and 9.1, 19 of up to 1801 with 31 queries 71.5, 60.4, 52.6 and 54.6.)
constexpr int WARPS = 4, TILE = 16, START = 24;
constexpr float SLACK = 4.f;       // powers of two by which a score may exceed the maximum that is kept
// Powers of two that the largest weight is held at: fp16 has numbers from 2^-24 to 2^16, and thousands of tokens with 2^-26 of the
// largest weight count together.
template <typename T>
constexpr float LIFT = std::is_same<T, __half>::value ? 11.f : 0.f;
using Cut = Runs<TILE, START, WARPS>;

struct AttnArgs {
  Cache c;
  const int* lengths;
  const void* q;
  void* out;
  float* lse;                 // [rows][heads][S] or nullptr
  float* weights;             // [rows][kv heads][places] or nullptr
  float* partial;             // sums [2 ctas][columns of a tile][D], then maximum and denominators [2 ctas][columns][4]
  int2* owners;               // first and last block of each [row][head and column tile]
  float* scores;              // [rows][kv heads][places of the table][columns], in powers of two, where there are weights
  float* lse2;                // [rows][kv heads][columns], the same
  long long places, q_batch, q_token; // (strides of q: elements)
  int S, heads, group;
  float scale_log2;           // softmax scale * log2(e)
  int ctas;                   // blocks that the work is cut for; 0: a block takes whole sequences (of a head), one after another
  int* status;
};

template <typename T>
ATB_DEVICE void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
ATB_DEVICE void ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
ATB_DEVICE void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
ATB_DEVICE uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(a, b);
  }
}
// whether one of two 16-bit numbers is an infinity or a NaN
template <typename T>
ATB_DEVICE bool endless(uint32_t u) {
  constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (u & E) == E || (u >> 16 & E) == E;
}

// Four dims of a column's result, from its maximum, the sum of its weights, that of the rounded ones, and the sums with the values.
template <typename T, int D>
ATB_DEVICE void finish(const AttnArgs& a, int b, int head, int n, int d, float top, float sum, float rounded, const float (&o)[4]) {
  const int i = n / a.group, h = head * a.group + n - i * a.group;
  const float inv = rounded == 0.f ? 0.f : 1.f / rounded;
  T y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(o[e] * inv);
  *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + (((long long)b * a.S + i) * a.heads + h) * D + d) =
      *reinterpret_cast<const uint2*>(y);
  if (d != 0) return;
  const float lse2 = top + (log2f(sum) - LIFT<T>);
  if (a.lse) a.lse[((long long)b * a.heads + h) * a.S + i] = lse2 * 0.69314718056f;
  if (a.lse2) a.lse2[((long long)b * a.c.kv_heads + head) * (a.S * a.group) + n] = lse2;
}

// Both products run on the warp's matrix instruction (16 x 8 x 16, fp32 sums), with the keys and the values as its 16-row operand
// and the columns as its 8-wide one: s[t, n] = k[t] . q[n], o[d, n] = sum_t v[t, d] p[t, n]. So a group of up to 8 query heads fills it.
// A tile of 16 tokens lies in one page; the copy unit brings its keys and values into a ring of the warp's own, STAGES tiles ahead, in
// halves of 64 dims whose rows are 128 bytes, their 16-byte pieces exchanged by the row (the 128-byte swizzle), so that a matrix load
// of 8 rows meets no bank twice.
// Weights p are rounded to the cache's 16 bits for their product with the values; what divides the sums is the sum of the rounded
// weights (a product with ones), so that they add up to 1, and the logarithm of the denominator comes from the unrounded ones.
// Scores are taken relative to the running maximum, which may be exceeded by 2^SLACK before everything is rescaled; only tiles at a
// sequence's end are masked. There, what no column sees is put to 0 in shared memory (memory behind a sequence may hold anything), and
// a value that some columns see and others do not is kept from the others even if it is an infinity or a NaN: column by column then.
// Bound by memory: two sequences of 100k tokens, 32 query heads on 8 of 128 (781 MB), 128 us, 6.1 TB/s; 32 of up to 4096 (241 MB) 45 us;
// one of 1531, 16 heads, 9.3. No tcgen05: with 1 to 32 columns the products take a fifth of the issue slots, and a detour through tensor
// memory would add to a segment's start and end; 31 queries of 4 heads (124 columns, 19 sequences) take 43 us and would gain from it.
template <int D, int NT>
struct Shape {
  static constexpr int COLS = 8 * NT, STAGE = TILE * D * 4, STAGES = 3 * 128 / D, RING = WARPS * STAGES * STAGE;
  static constexpr int QUERIES = NT == 4 ? COLS * D * 2 : 0;      // bytes of shared memory for them; else they lie in registers
  static constexpr int SMEM = RING + QUERIES + 1024, BLOCKS = 2;  // of an SM; the ring begins on 1024 bytes
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(WARPS * 32, Shape<D, NT>::BLOCKS) kv_attention_kernel(const __grid_constant__ CUtensorMap map, AttnArgs a) {
  using Sh = Shape<D, NT>;
  constexpr int KS = D / 16, COLS = Sh::COLS, STAGES = Sh::STAGES, HALF_BYTES = TILE * 128;
  constexpr uint32_t ONES = std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u;
  static_assert(WARPS * COLS * (D + 4) * 4 <= Sh::RING, "the warps' sums lie in the place of the ring");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ float sh_m[WARPS][COLS], sh_l[WARPS][COLS], sh_r[WARPS][COLS];
  __shared__ uint64_t bars[WARPS][STAGES];
  __shared__ int abort_flag;
  const Cache& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, q4 = lane & 3;
  uint8_t* const ring = smem + warp * (STAGES * Sh::STAGE);
  uint32_t* const sh_q = reinterpret_cast<uint32_t*>(smem + Sh::RING);
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane < STAGES) mbar_init(&bars[warp][lane], 1);
  mbar_fence_init();
  if (threadIdx.x == 0) tma_prefetch_desc(&map);
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
  uint32_t stage_in = 0, stage_out = 0, phase_out = 0;       // of the warp's ring: where the next tile goes, the next one comes from

  // where a lane reads its row of a matrix load in a half of a tile: keys (tokens 0..7, 8..15, then the next 8 dims) and values (the
  // next 8 dims, then tokens 8..15)
  const uint32_t k_row = (lane & 15) * 128, k_piece = lane >> 4, v_row = ((lane >> 4) * 8 + (lane & 7)) * 128, v_piece = (lane >> 3) & 1;
  const uint32_t turn = lane & 7, ring_at = smem_u32(ring);

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

    // pages of the warp's tiles j to j + 31
    auto pages_from = [&](int j) {
      const int t = (t_first + warp + (j + lane) * WARPS) * TILE;
      int page = 0;
      if (j + lane < mine) {
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
      if (j > 0 && (j & 31) == 0) pages = pages_from(j);
      const int page = __shfl_sync(0xffffffffu, pages, j & 31);
      const int t = (t_first + warp + j * WARPS) * TILE;
      if (lane == 0) mbar_expect_tx(&bars[warp][stage_in], Sh::STAGE);
      __syncwarp();
      if (lane < 2)
        tma_load_3d(ring + stage_in * Sh::STAGE + lane * (Sh::STAGE / 2), &map, &bars[warp][stage_in], 0,
                    (((page * 2 + lane) * c.kv_heads + head) << c.page_shift) + (t & ((1 << c.page_shift) - 1)), 0);
      stage_in = stage_in + 1 == STAGES ? 0 : stage_in + 1;
    };
    for (int j = 0; j < STAGES; ++j) fetch(j);

    // queries: of column 8 j + r the dims 16 k + 2 q4, + 1 and 8 further
    uint32_t qf[NT == 4 ? 1 : NT][KS][2];
    auto query = [&](int n) {
      const bool live = n < columns;
      const int i = live ? n / a.group : 0, h = live ? n - i * a.group : 0;
      return live ? reinterpret_cast<const T*>(a.q) + b * a.q_batch + i * a.q_token + (long long)(head * a.group + h) * D : nullptr;
    };
    if constexpr (NT == 4) {
      // [k][lane][8 words]: those of four column tiles side by side
      for (int x = threadIdx.x; x < KS * 32 * 4; x += WARPS * 32) {
        const int j = x & 3, l = x >> 2 & 31, k = x >> 7;
        const T* q = query(col_tile * COLS + 8 * j + (l >> 2));
        uint2 w = make_uint2(0u, 0u);
        if (q) {
          w.x = *reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * (l & 3));
          w.y = *reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * (l & 3) + 8);
        }
        *reinterpret_cast<uint2*>(sh_q + (k * 32 + l) * 8 + 2 * j) = w;
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const T* q = query(col_tile * COLS + 8 * j + r);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) qf[j][k][e] = q ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * q4 + 8 * e) : 0u;
      }
    }
    // the keys that columns 8 j + 2 q4 + {0, 1} see, and that all of the tile see
    int limit[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int o = 0; o < 2; ++o) limit[j][o] = min(len, len - a.S + (col_tile * COLS + 8 * j + 2 * q4 + o) / a.group + 1);
    const int all_see = len - a.S + col_tile * COLS / a.group + 1;
    float* const scores = a.scores ? a.scores + ((long long)b * c.kv_heads + head) * ((long long)c.width << c.page_shift) * columns : nullptr;

    // running maximum of the scores (m), sums of p (l), of its rounded values (ones), and with the values; `ref` is what scores are
    // taken relative to: m - LIFT, or 0 where there is none yet
    float o_acc[NT][KS][4], ones[NT][4], m[NT][2], ref[NT][2], l[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o_acc[j][i][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) ones[j][e] = 0.f;
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        m[j][o] = -INFINITY;
        ref[j][o] = l[j][o] = 0.f;
      }
    }
    bool unset = true;     // whether a column has no maximum yet

    auto tile = [&](uint32_t keys, int t0, auto masked) {
      constexpr bool MASK = decltype(masked)::value;
      const uint32_t values = keys + Sh::STAGE / 2;
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t x[4];
        ldmatrix(x, keys + (k >> 2) * HALF_BYTES + k_row + (((2 * (k & 3) + k_piece) ^ turn) << 4));
        if constexpr (NT == 4) {
          const uint4 u0 = *reinterpret_cast<const uint4*>(sh_q + (k * 32 + lane) * 8), u1 = *reinterpret_cast<const uint4*>(sh_q + (k * 32 + lane) * 8 + 4);
          mma_16<T>(s[0], x, u0.x, u0.y);
          mma_16<T>(s[1], x, u0.z, u0.w);
          mma_16<T>(s[2], x, u1.x, u1.y);
          mma_16<T>(s[3], x, u1.z, u1.w);
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16<T>(s[n], x, qf[n][k][0], qf[n][k][1]);
        }
      }
      float over = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int o = e & 1, t = t0 + r + 4 * (e & 2);
          float v = s[n][e] * a.scale_log2;
          if (MASK && t >= limit[n][o]) v = -INFINITY;
          s[n][e] = v;
        }
      if (scores) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int col = col_tile * COLS + 8 * n + 2 * q4, t = t0 + r + 8 * i;
            if (MASK && t >= len) continue;
            float* const dst = scores + (long long)t * columns + col;
            if (columns % 2 == 0) {
              if (col < columns) *reinterpret_cast<float2*>(dst) = make_float2(s[n][2 * i], s[n][2 * i + 1]);
            } else {
              if (col < columns) dst[0] = s[n][2 * i];
              if (col + 1 < columns) dst[1] = s[n][2 * i + 1];
            }
          }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] -= ref[n][e & 1];
          over = fmaxf(over, s[n][e]);
        }
      if (__any_sync(0xffffffffu, over > SLACK + LIFT<T> || unset)) {
        unset = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float f[2];
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            float most = fmaxf(s[n][o], s[n][2 + o]);
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, k));
            const float to = fmaxf(m[n][o], ref[n][o] + most), by = to == -INFINITY ? 0.f : to - LIFT<T> - ref[n][o];
            f[o] = m[n][o] == -INFINITY ? (l[n][o] == 0.f ? 0.f : 1.f) : fast_exp2(-by);
            m[n][o] = to;
            ref[n][o] += by;
            unset = unset || to == -INFINITY;
            l[n][o] *= f[o];
            s[n][o] -= by;
            s[n][2 + o] -= by;
          }
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o_acc[n][i][e] *= f[e & 1];
#pragma unroll
          for (int e = 0; e < 4; ++e) ones[n][e] *= f[e & 1];
        }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float w0 = fast_exp2(s[n][2 * i]), w1 = fast_exp2(s[n][2 * i + 1]);
          l[n][0] += w0;
          l[n][1] += w1;
          pf[n][i] = transpose_8x8(pack2<T>(w0, w1));
        }
      const uint32_t one[4] = {ONES, ONES, ONES, ONES};
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_16<T>(ones[n], one, pf[n][0], pf[n][1]);
      if constexpr (MASK) {
        // values from row `from` on become 0
        auto clear = [&](int from) {
          for (int x = lane; x < 2 * (D / 64) * 4 * TILE; x += 32) {
            const int t = x % TILE, piece = x / TILE;
            if (t >= from)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(values + (piece >> 3) * HALF_BYTES + t * 128 + (piece & 7) * 16), "r"(0u) : "memory");
          }
          __syncwarp();
        };
        clear(len - t0);
        bool odd = false;      // an infinity or a NaN that some columns do not see
        if (a.S > 1)
          for (int x = lane; x < 2 * (D / 64) * 4 * TILE; x += 32) {
            const int t = x % TILE, piece = x / TILE;
            if (t0 + t >= all_see) {
              uint32_t w[4];
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(values + (piece >> 3) * HALF_BYTES + t * 128 + (piece & 7) * 16) : "memory");
              odd = odd || endless<T>(w[0]) || endless<T>(w[1]) || endless<T>(w[2]) || endless<T>(w[3]);
            }
          }
        if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
          for (int n = NT - 1; n >= 0; --n)
#pragma unroll 1
            for (int col = 7; col >= 0; --col) {
              clear(len - a.S + (col_tile * COLS + 8 * n + col) / a.group + 1 - t0);
              const uint32_t p0 = r == col ? pf[n][0] : 0u, p1 = r == col ? pf[n][1] : 0u;
#pragma unroll
              for (int i = 0; i < KS; ++i) {
                uint32_t y[4];
                ldmatrix_trans(y, values + (i >> 2) * HALF_BYTES + v_row + (((2 * (i & 3) + v_piece) ^ turn) << 4));
                float z[4] = {0.f, 0.f, 0.f, 0.f};
                mma_16<T>(z, y, p0, p1);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (2 * q4 + (e & 1) == col) o_acc[n][i][e] += z[e];
              }
            }
          fence_proxy_async_smem();
          return;
        }
        fence_proxy_async_smem();        // the copy unit writes here next
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        uint32_t y[4];
        ldmatrix_trans(y, values + (i >> 2) * HALF_BYTES + v_row + (((2 * (i & 3) + v_piece) ^ turn) << 4));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_16<T>(o_acc[n][i], y, pf[n][0], pf[n][1]);
      }
    };

    bool arrived = true;
    for (int j = 0; j < mine; ++j) {
      const int t0 = (t_first + warp + j * WARPS) * TILE;
      arrived = mbar_wait_warp(&bars[warp][stage_out], phase_out, &abort_flag, a.status);
      if (!arrived) break;
      if (t0 + TILE <= all_see) tile(ring_at + stage_out * Sh::STAGE, t0, std::false_type());
      else tile(ring_at + stage_out * Sh::STAGE, t0, std::true_type());
      if (++stage_out == STAGES) {
        stage_out = 0;
        phase_out ^= 1;
      }
      __syncwarp();
      fetch(j + STAGES);
    }

    // the warps' sums, in their order, in the place of the rings: every copy has arrived and been read
    float (*const sh_o)[COLS][D + 4] = reinterpret_cast<float (*)[COLS][D + 4]>(smem);
    if (__syncthreads_or(!arrived)) {
      // a copy did not come in time: nothing more is asked for or stored, and those on their way may land before the block ends
      const uint64_t t_start = globaltimer_ns();
      while (globaltimer_ns() - t_start < 200000ull) __nanosleep(1000);
      return;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int o = 0; o < 2; ++o) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) l[j][o] += __shfl_xor_sync(0xffffffffu, l[j][o], k);
        const int col = 8 * j + 2 * q4 + o;
        if (r == 0) {
          sh_m[warp][col] = m[j][o];
          sh_l[warp][col] = l[j][o];
          sh_r[warp][col] = ones[j][o];
        }
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          sh_o[warp][col][16 * i + r] = o_acc[j][i][o];
          sh_o[warp][col][16 * i + r + 8] = o_acc[j][i][2 + o];
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
      float sum = 0.f, rounded = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float f = sh_m[k][col] == -INFINITY ? (sh_l[k][col] == 0.f ? 0.f : 1.f) : fast_exp2(sh_m[k][col] - top);
        const float4 v = *reinterpret_cast<const float4*>(&sh_o[k][col][d]);
        sum += f * sh_l[k][col];
        rounded += f * sh_r[k][col];
        o[0] += f * v.x;
        o[1] += f * v.y;
        o[2] += f * v.z;
        o[3] += f * v.w;
      }
      if (!whole) {
        *reinterpret_cast<float4*>(a.partial + (slot * COLS + col) * D + d) = make_float4(o[0], o[1], o[2], o[3]);
        if (d == 0)
          *reinterpret_cast<float4*>(a.partial + 2LL * a.ctas * COLS * D + (slot * COLS + col) * 4) = make_float4(top, sum, rounded, 0.f);
      } else {
        finish<T, D>(a, b, head, n, d, top, sum, rounded, o);
      }
    }
    if (u < run_end) {
      fence_proxy_async_smem();      // the sums were written by the threads, the next tiles come by the copy unit
      __syncthreads();
    }
  }
}

// Maximum and sums of a column of a sequence that several blocks worked on, and with V its four dims from d: the blocks' results are read
// eight at a time, independent of one another, and joined in the order of the blocks.
template <int D, int COLS, bool V>
ATB_DEVICE void join_column(const AttnArgs& a, int2 own, int col, int d, float& top, float& sum, float& rounded, float (&o)[4]) {
  constexpr int EACH = 8;
  const float* const stats = a.partial + 2LL * a.ctas * COLS * D;
  top = -INFINITY;
  sum = rounded = o[0] = o[1] = o[2] = o[3] = 0.f;
  for (int k0 = own.x; k0 <= own.y; k0 += EACH) {
    float4 ml[EACH], v[V ? EACH : 1];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const long long at = (2LL * min(k0 + k, own.y) + (k0 + k == own.x)) * COLS + col;
      ml[k] = *reinterpret_cast<const float4*>(stats + 4 * at);
      if constexpr (V) v[k] = *reinterpret_cast<const float4*>(a.partial + at * D + d);
      if (k0 + k > own.y) ml[k] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    }
    float to = top;
#pragma unroll
    for (int k = 0; k < EACH; ++k) to = fmaxf(to, ml[k].x);
    const float down = top == -INFINITY ? (sum == 0.f ? 0.f : 1.f) : fast_exp2(top - to);
    sum *= down;
    rounded *= down;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= down;
    top = to;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      if (k0 + k > own.y) continue;
      const float f = ml[k].x == -INFINITY ? (ml[k].y == 0.f ? 0.f : 1.f) : fast_exp2(ml[k].x - top);
      sum += f * ml[k].y;
      rounded += f * ml[k].z;
      if constexpr (V) {
        o[0] += f * v[k].x;
        o[1] += f * v[k].y;
        o[2] += f * v[k].z;
        o[3] += f * v[k].w;
      }
    }
  }
}
ATB_DEVICE bool shared_by_blocks(const AttnArgs& a, int2 own) {       // (behind a kernel that left early there may be anything)
  return own.x >= 0 && own.y < a.ctas && own.x < own.y;
}
// The join of one sequence, head and column tile (a block). Bound by latency.
template <typename T, int D, int NT>
ATB_DEVICE void join(const AttnArgs& a, int item, int per) {
  constexpr int COLS = 8 * NT;
  const int2 own = a.owners[item];
  if (!shared_by_blocks(a, own)) return;
  const int columns = a.S * a.group, b = item / per, hc = item - b * per;
  const int head = hc % a.c.kv_heads, col_tile = hc / a.c.kv_heads;
  for (int x = threadIdx.x; x < COLS * (D / 4); x += 256) {
    const int col = x / (D / 4), d = (x - col * (D / 4)) * 4, n = col_tile * COLS + col;
    if (n >= columns) continue;
    float top, sum, rounded, o[4];
    join_column<D, COLS, true>(a, own, col, d, top, sum, rounded, o);
    finish<T, D>(a, b, head, n, d, top, sum, rounded, o);
  }
}
template <typename T, int D, int NT>
__global__ void __launch_bounds__(256) kv_join_kernel(AttnArgs a, int per) {
  grid_go();
  grid_wait();
  if (__syncthreads_or(*a.status != 0)) return;
  join<T, D, NT>(a, blockIdx.x, per);
}

// What the queries attended to: a place's scores of all columns, as the kernel above has left them, relative to the columns' logarithms,
// added up by LANES lanes in one order, and to what is there. Logarithms of sequences that several blocks worked on are
// joined here, MOST columns at a time; the last blocks of a head's row do the join of the results beside it. Bound by latency: reads of
// blocks' results, scores and sums one after another (16 sequences of 1152, 32 heads: 5 us with the join, 8 in two launches).
template <typename T, int D, int NT, int LANES>
__global__ void __launch_bounds__(256, 3) kv_weights_kernel(AttnArgs a, int per, int chunks) {
  constexpr int COLS = 8 * NT, MOST = 128;
  __shared__ float lse2[MOST];
  grid_go();
  grid_wait();
  const Cache& c = a.c;
  const int columns = a.S * a.group, b = blockIdx.x / c.kv_heads, head = blockIdx.x - b * c.kv_heads, lane = threadIdx.x % LANES;
  const bool failed = threadIdx.x == 0 && *a.status != 0;
  const int len = seen_length(c, a.lengths, b, a.status);
  if (__syncthreads_or(failed)) return;
  if ((int)blockIdx.y >= chunks) {
    join<T, D, NT>(a, b * per + ((int)blockIdx.y - chunks) * c.kv_heads + head, per);
    return;
  }
  const float* const scores = a.scores + (long long)blockIdx.x * ((long long)c.width << c.page_shift) * columns;
  float* const weights = a.weights + (long long)blockIdx.x * a.places;
  const int step = chunks * (256 / LANES);
  for (int n0 = 0; n0 < columns; n0 += MOST) {
    const int n1 = min(columns - n0, MOST);
    __syncthreads();
    if ((int)threadIdx.x < n1) {
      const int n = n0 + threadIdx.x, col_tile = n / COLS;
      const int2 own = a.ctas > 0 ? a.owners[(long long)b * per + col_tile * c.kv_heads + head] : make_int2(0, 0);
      float x;
      if (shared_by_blocks(a, own)) {
        float top, sum, rounded, o[4];
        join_column<D, COLS, false>(a, own, n - col_tile * COLS, 0, top, sum, rounded, o);
        x = top + (log2f(sum) - LIFT<T>);
      } else {
        x = a.lse2[(long long)blockIdx.x * columns + n];
      }
      lse2[threadIdx.x] = x;
    }
    __syncthreads();
    // (several places of a thread at once: their scores and what is there are on their way together)
    constexpr int U = LANES == 1 ? 4 : 2, C = LANES == 1 ? 4 : 16;       // C LANES columns in a go
    for (int t0 = blockIdx.y * (256 / LANES) + threadIdx.x / LANES; t0 - (int)threadIdx.x / LANES < len; t0 += U * step) {
      float x[U][C], old[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * step;
        old[u] = t < len ? weights[t] : 0.f;
#pragma unroll
        for (int k = 0; k < C; ++k) x[u][k] = t < len && lane + k * LANES < n1 ? scores[(long long)t * columns + n0 + lane + k * LANES] : -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * step;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < C; ++k) {
          const float y = lane + k * LANES < n1 ? lse2[lane + k * LANES] : -INFINITY;
          sum += x[u][k] == -INFINITY || y == -INFINITY ? 0.f : fast_exp2(x[u][k] - y);
        }
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (t < len && lane == 0) weights[t] = old[u] + sum;
      }
    }
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
  int* first;                 // [units] the first place whose token changes, `budget` where none does, WRONG where nothing may
  int* source;                // [units][budget] place in the pool (page, slot) of the token that a place takes
  float* kept;                // [units][budget] its weight
  long long places, layer_elements;
  int budget, recent, layers;
  int* status;
};
// A sequence that is longer than its row of the page table, or whose pages are not all there, is left as it is. That is found by the
// selection, and recorded by the move: within a launch nobody changes the status word that says whether to begin.
constexpr int WRONG = -1;
// A number whose order as an unsigned integer is that of f; both zeros alike, a NaN as -inf.
ATB_DEVICE uint32_t rank_of(float f) {
  const uint32_t u = __float_as_uint((f != f ? -INFINITY : f) + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Sum of v over the threads before this one, and over all; `red` is a shared int[32].
ATB_DEVICE int block_before(int v, int* red, int& all) {
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
  const int x = lane < warps ? red[lane] : 0;
  int up = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += y;
  }
  all = __shfl_sync(0xffffffffu, up, 31);
  return __shfl_sync(0xffffffffu, up - x, w) + sum - v;
}

// What a unit (a key/value head of a sequence in a layer) keeps: the blocks of a cluster have a share of its places each. The least
// rank that is kept is found digit by digit, 8 bits at a time, from counts that the blocks read from each other's shared memory, until
// so few are left that each is compared with each; of the places of that rank the lowest are kept. Then the places that are kept are
// numbered in their order: that number is where the token goes. Weights are moved through the workspace, so that no block writes what
// another still reads. Bound by latency: reads of lengths, pages and weights one after another, a few meetings of the block (512 units of
// up to 1152 places 15 us, 8 of 100003 by eight blocks each 40).
constexpr int BINS = 256, EACH = 4, FEW = 256;
template <int SELECT>
__global__ void __launch_bounds__(SELECT) kv_select_kernel(EvictArgs a, int room) {
  extern __shared__ __align__(16) float sh_w[];   // `room` weights of the share; the others are read again
  __shared__ int hist[3][BINS], red[32], sh_digit, sh_above, sh_in, sh_counts[2], sh_least, sh_failed, sh_n;
  __shared__ uint32_t few[FEW], few_all[FEW], sh_rank;
  cg::cluster_group cluster = cg::this_cluster();
  for (int i = threadIdx.x; i < 3 * BINS; i += SELECT) hist[0][i] = 0;
  grid_go();
  grid_wait();
  const Cache& c = a.c;
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const long long unit = blockIdx.x / blocks;
  const int b = (int)(unit / c.kv_heads % c.rows);
  auto meet = [&] {
    if (blocks == 1) __syncthreads();
    else cluster.sync();
  };
  const int before = threadIdx.x == 0 ? *a.status : 0;       // on its way beside the lengths
  const int len = a.lengths[b], lane = threadIdx.x & 31;
  const bool leader = rank == 0 && threadIdx.x == 0, too_long = len > c.width << c.page_shift;
  if (leader && unit < (long long)c.rows * c.kv_heads && unit % c.kv_heads == 0) a.out[b] = too_long ? len : min(len, a.budget);
  if (len <= a.budget || too_long) {
    if (leader) a.first[unit] = too_long ? WRONG : a.budget;
    return;
  }
  const int part = (((len + blocks - 1) / blocks + 3) & ~3), from = min(len, rank * part), to = min(len, from + part);
  float* const w = a.weights + unit * a.places;
  const int held = min(to - from, room);
#pragma unroll 16
  for (int i = threadIdx.x; i < held; i += SELECT) sh_w[i] = w[from + i];
  bool bad = false;
  for (int i = (from >> c.page_shift) + threadIdx.x; i << c.page_shift < to; i += SELECT) bad = bad || page_of(c, b, i << c.page_shift) < 0;
  if (threadIdx.x == 0) {
    sh_least = len;
    sh_failed = before != 0;
    sh_n = 0;
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0 && bad) sh_failed |= 2;
  auto weight = [&](int i) { return i - from < held ? sh_w[i - from] : w[i]; };

  const int n = len - a.recent, mine = min(to, n);      // those from n on stay
  int left = a.budget - a.recent;            // of rank `least`, so many are kept
  uint32_t least = left == 0 ? 0xffffffffu : 0u;
  int failed = 0;
  int shift = 32;                            // digits above this are known
#pragma unroll 1
  for (int pass = 0; shift > 0; ++pass) {
    shift -= 8;
    int* const h = hist[pass % 3];
    if (left > 0) {
#pragma unroll 4
      for (int i0 = from; i0 < mine; i0 += SELECT) {
        const int i = i0 + threadIdx.x;
        const uint32_t r = i < mine ? rank_of(weight(i)) : 0u;
        const bool in = i < mine && (pass == 0 || (r ^ least) >> (shift + 8) == 0);
        const int bin = in ? (int)(r >> shift & (BINS - 1)) : -1;
        int same;
        __match_all_sync(0xffffffffu, bin, &same);       // (many weights alike would wait for one another)
        if (!same) {
          if (in) atomicAdd(&h[bin], 1);
        } else if (in && lane == 0) {
          atomicAdd(&h[bin], 32);
        }
      }
    }
    meet();
    if (pass == 0)
      for (int i = 0; i < blocks; ++i) failed |= *cluster.map_shared_rank(&sh_failed, i);
    if (pass == 1 && threadIdx.x < BINS) hist[0][threadIdx.x] = 0;       // the first digit's counts have been read by all
    if (left > 0 && !failed) {
      // from the highest bin down: one of a thread
      static_assert(BINS <= SELECT, "a thread has a bin");
      const int digit = BINS - 1 - (int)threadIdx.x;
      int count = 0, all;
      if (digit >= 0)
        for (int i = 0; i < blocks; ++i) count += cluster.map_shared_rank(h, i)[digit];
      const int above = block_before(count, red, all);
      if (above < left && above + count >= left) {
        sh_digit = digit;
        sh_above = above;
        sh_in = count;
      }
      __syncthreads();
      least |= (uint32_t)sh_digit << shift;
      left -= sh_above;
      if (sh_in <= FEW && shift > 0) {
        // few with these digits: every block gets the ranks of all, and finds the left-th largest
#pragma unroll 4
        for (int i = from + threadIdx.x; i < mine; i += SELECT) {
          const uint32_t r = rank_of(weight(i));
          if ((r ^ least) >> shift == 0) few[atomicAdd(&sh_n, 1)] = r;
        }
        meet();
        const int theirs = lane < blocks ? *cluster.map_shared_rank(&sh_n, lane) : 0, total = __reduce_add_sync(0xffffffffu, theirs);
        const int r_of = threadIdx.x >> 5;       // a warp for each block
        int at = 0;
        for (int i = 0; i < blocks; ++i) {
          const int m = __shfl_sync(0xffffffffu, theirs, i);
          if (i < r_of) at += m;
        }
        if (r_of < blocks) {
          const uint32_t* const other = cluster.map_shared_rank(few, r_of);
          const int m = __shfl_sync(0xffffffffu, theirs, r_of);
          for (int i = lane; i < m; i += 32) few_all[at + i] = other[i];
        }
        __syncthreads();
        if ((int)threadIdx.x < total) {
          const uint32_t r = few_all[threadIdx.x];
          int greater = 0, same = 0;
#pragma unroll 4
          for (int i = 0; i < total; ++i) {
            greater += few_all[i] > r;
            same += few_all[i] == r;
          }
          if (greater < left && greater + same >= left) {      // (all that are alike say the same)
            sh_rank = r;
            sh_above = greater;
          }
        }
        __syncthreads();
        least = sh_rank;
        left -= sh_above;
        shift = 0;
      }
    }
    __syncthreads();
  }
  // places above and at the border, before the share
  int all, above_before = 0, ties_before = 0;
  if (blocks > 1) {
    int above = 0, ties = 0;
#pragma unroll 4
    for (int i = from + threadIdx.x; i < to; i += SELECT) {
      const uint32_t r = rank_of(weight(i));
      above += i >= n || r > least;
      ties += i < n && r == least;
    }
    block_before(above, red, all);
    if (threadIdx.x == 0) sh_counts[0] = all;
    block_before(ties, red, all);
    if (threadIdx.x == 0) sh_counts[1] = all;
    cluster.sync();
    for (int i = 0; i < rank; ++i) {
      above_before += cluster.map_shared_rank(sh_counts, i)[0];
      ties_before += cluster.map_shared_rank(sh_counts, i)[1];
    }
  }
  if (!failed) {
    int* const source = a.source + unit * a.budget;
    float* const kept = a.kept + unit * a.budget;
    int first = len, page = from + (int)threadIdx.x * EACH < to ? page_of(c, b, from + threadIdx.x * EACH) : 0;
    for (int i0 = from; i0 < to; i0 += SELECT * EACH) {
      const int i1 = i0 + threadIdx.x * EACH;
      const int next = i1 + SELECT * EACH < to ? page_of(c, b, i1 + SELECT * EACH) : 0;       // (pages have a multiple of EACH places)
      float f[EACH];
      if (i1 - from + EACH <= held) {       // (the share begins on a multiple of EACH)
        const float4 v = *reinterpret_cast<const float4*>(sh_w + (i1 - from));
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < EACH; ++e) f[e] = i1 + e < to ? weight(i1 + e) : 0.f;
      }
      int count = 0;                        // above in the low half, ties in the high one
      bool is_above[EACH], is_tie[EACH];
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = i1 + e;
        const uint32_t r = rank_of(f[e]);
        is_above[e] = i < to && (i >= n || r > least);
        is_tie[e] = i < to && i < n && r == least;
        count += is_above[e] + (is_tie[e] << 16);
      }
      const int before_me = block_before(count, red, all);
      int g = above_before + (before_me & 0xffff), t = ties_before + (before_me >> 16);
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = i1 + e;
        if (is_above[e] || (is_tie[e] && t < left)) {
          const int at = g + min(t, left);
          source[at] = (page << c.page_shift) + (i & ((1 << c.page_shift) - 1));
          kept[at] = f[e];
        } else if (i < to) {
          first = min(first, i);
        }
        g += is_above[e];
        t += is_tie[e];
      }
      above_before += all & 0xffff;
      ties_before += all >> 16;
      page = next;
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) atomicMin(&sh_least, first);
  }
  meet();
  if (leader) {
    int first = len;
    for (int i = 0; i < blocks; ++i) first = min(first, *cluster.map_shared_rank(&sh_least, i));
    a.first[unit] = failed & 2 ? WRONG : failed ? a.budget : min(first, a.budget);
  }
  if (!failed) {
    const float* const kept = a.kept + unit * a.budget;
#pragma unroll 16
    for (int i = from + threadIdx.x; i < to; i += SELECT) w[i] = i < a.budget ? kept[i] : 0.f;
  }
  if (blocks > 1) cluster.sync();                // the first has read the others' words
}

// The tokens' move: a block has the keys or the values of a unit and takes places in their order, THREADS PER pieces of 16 bytes in a
// round. A token only moves down, so what a place's token comes from is not written before that place's turn: the reads of a round end
// before its writes begin, and those of later rounds may come before either. Bound by memory where there are many units (8 layers of 8
// sequences, 8 heads: 64 us for 406 MB).
template <int D, int THREADS, int PER>
__global__ void __launch_bounds__(THREADS) kv_move_kernel(EvictArgs a) {
  grid_go();
  grid_wait();
  const Cache& c = a.c;
  const int which = blockIdx.x & 1;
  const long long unit = blockIdx.x / 2;
  const int first = a.first[unit];
  if (first == WRONG && threadIdx.x == 0) atomicCAS(a.status, 0, (int)ATB_ERR_BAD_INDEX);
  if (first == WRONG || first >= a.budget) return;
  const int head = (int)(unit % c.kv_heads), b = (int)(unit / c.kv_heads % c.rows), mask = (1 << c.page_shift) - 1;
  constexpr int LANES = D / 8, ROWS = THREADS / LANES, STEP = ROWS * PER;
  uint4* const data = reinterpret_cast<uint4*>((__half*)c.data + unit / c.kv_heads / c.rows * a.layer_elements) + threadIdx.x % LANES;
  const int* const source = a.source + unit * a.budget;
  const int* const row = c.table + b * c.table_stride;
  auto at = [&](int page, int slot) -> uint4* { return data + (((((long long)page * 2 + which) * c.kv_heads + head) << c.page_shift) + slot) * LANES; };
  int src[PER];
  auto ask = [&](int j0) {                 // where the round's rows come from
#pragma unroll
    for (int k = 0; k < PER; ++k) src[k] = j0 + k * ROWS < a.budget ? source[j0 + k * ROWS] : -1;
  };
  uint4 x[2][PER];
  auto load = [&](uint4 (&y)[PER]) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (src[k] >= 0) y[k] = *at(src[k] >> c.page_shift, src[k] & mask);
  };
  auto store = [&](const uint4 (&y)[PER], int j0) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int j = j0 + k * ROWS;
      if (j < a.budget) *at(row[j >> c.page_shift], j & mask) = y[k];
    }
  };
  const int own = threadIdx.x / LANES;
  ask(first + own);
  load(x[0]);
  ask(first + own + STEP);
  for (int j0 = first;; j0 += 2 * STEP) {  // (as many rounds for all threads)
    __syncthreads();
    load(x[1]);
    ask(j0 + own + 2 * STEP);
    store(x[0], j0 + own);
    if (j0 + STEP >= a.budget) break;
    __syncthreads();
    load(x[0]);
    ask(j0 + own + 3 * STEP);
    store(x[1], j0 + own + STEP);
    if (j0 + 2 * STEP >= a.budget) break;
  }
}

// The same for few units: the blocks of a cluster share the rows of a round. DEEP rounds are on their way in shared memory, and the blocks
// say that they have their part of the next round before they write this one, so that nobody waits for the meeting. 50000 tokens of 8
// heads (410 MB): 112 us, bound by the rounds' latency; meetings that wait, one round ahead, took 163, a slab of the rows' 32 bytes for
// every block, which need not meet, 108, for its many small requests.
template <int D, int THREADS, int PER, int DEEP>
__global__ void __launch_bounds__(THREADS) kv_move_cluster_kernel(EvictArgs a) {
  extern __shared__ uint4 ring[];          // [DEEP][PER][THREADS]: a thread reads what it has asked for itself
  cg::cluster_group cluster = cg::this_cluster();
  grid_go();
  grid_wait();
  const Cache& c = a.c;
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), which = blockIdx.x / blocks & 1;
  const long long unit = blockIdx.x / blocks / 2;
  const int first = a.first[unit];
  if (first == WRONG && threadIdx.x == 0) atomicCAS(a.status, 0, (int)ATB_ERR_BAD_INDEX);
  if (first == WRONG || first >= a.budget) return;
  const int head = (int)(unit % c.kv_heads), b = (int)(unit / c.kv_heads % c.rows), mask = (1 << c.page_shift) - 1;
  constexpr int LANES = D / 8, ROWS = THREADS / LANES;
  uint4* const data = reinterpret_cast<uint4*>((__half*)c.data + unit / c.kv_heads / c.rows * a.layer_elements) + threadIdx.x % LANES;
  const int* const source = a.source + unit * a.budget;
  const int* const row = c.table + b * c.table_stride;
  auto at = [&](int page, int slot) -> uint4* { return data + (((((long long)page * 2 + which) * c.kv_heads + head) << c.page_shift) + slot) * LANES; };
  const int own = rank * PER * ROWS + threadIdx.x / LANES, step = blocks * PER * ROWS;
  struct Sources {
    int at[PER];
  };
  auto ask = [&](int j0) {                 // where the round's rows come from
    Sources s;
#pragma unroll
    for (int k = 0; k < PER; ++k) s.at[k] = j0 + own + k * ROWS < a.budget ? source[j0 + own + k * ROWS] : -1;
    return s;
  };
  auto load = [&](int stage, const Sources& s) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (s.at[k] >= 0)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(ring + (stage * PER + k) * THREADS + threadIdx.x)),
                     "l"(__cvta_generic_to_global(at(s.at[k] >> c.page_shift, s.at[k] & mask))) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // What the meeting orders are reads that have come, before writes that other blocks then make. Only release and acquire say so; the
  // release also waits for this thread's writes of the round before (50001 of 100003 tokens, 8 heads: 158 us with the selection, 146 with
  // a relaxed arrival, which promises no order).
  auto arrive = [] { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); };
  Sources next = ask(first), far = ask(first + step);
  for (int s = 0; s < DEEP; ++s) {
    load(s, next);
    next = far;
    far = ask(first + (s + 2) * step);
  }
  asm volatile("cp.async.wait_group %0;" ::"n"(DEEP - 1) : "memory");
  arrive();
  cluster.barrier_wait();
  int stage = 0;
  for (int j0 = first; j0 < a.budget; j0 += step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(DEEP - 2) : "memory");      // the next round is here
    arrive();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int j = j0 + own + k * ROWS;
      if (j < a.budget) *at(row[j >> c.page_shift], j & mask) = ring[(stage * PER + k) * THREADS + threadIdx.x];
    }
    load(stage, next);                     // of the round DEEP further on; an empty group behind the last one
    next = far;
    far = ask(j0 + (DEEP + 2) * step);
    stage = stage + 1 == DEEP ? 0 : stage + 1;
    cluster.barrier_wait();
  }
}

// A budget that no sequence can be over: the lengths as they are.
__global__ void __launch_bounds__(256) kv_lengths_kernel(EvictArgs a) {
  grid_go();
  grid_wait();
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < a.c.rows) {
    seen_length(a.c, a.lengths, b, a.status);
    a.out[b] = a.lengths[b];
  }
}

Cache cache_of(void* data, const void* table, long long table_stride, int rows, int width, int pages, int kv_heads, int page_shift) {
  return Cache{{(const int*)table, table_stride, rows, width, pages, kv_heads, page_shift}, data};
}

template <typename T, int D>
int launch_append(const void* qkv, void* q, void* k, const Cache& c, const void* seq, const void* pos, const void* angles,
                  const void* cosT, const void* sinT, int positions, int tokens, int n_q, long long stride, cudaStream_t st, int* status) {
  const int each = SMALL / (D / 16), heads = n_q + 2 * c.kv_heads;
  // where there are more blocks than the GPU holds, a thread has three heads: more loads on their way, one look at the page table and the
  // angles
  const bool many = (long long)tokens * ((heads + each - 1) / each) > 148 * 16 && heads > each;
  const int blocks = many ? (heads + 3 * each - 1) / (3 * each) : (heads + each - 1) / each;
  if (blocks > 65535) return -2;
  return launched(launch_after(many ? kv_append_kernel<T, D, 3> : kv_append_kernel<T, D, 1>, dim3(tokens, blocks), SMALL, 0, st, 1,
                               (const T*)qkv, (T*)q, (T*)k, c, (const int*)seq, (const int*)pos, (const int*)angles, (const float*)cosT,
                               (const float*)sinT, positions, n_q, stride, status));
}

// The cache's rows of D as rows of 64: boxes of TILE rows of all D dims, the halves one behind another.
template <int D>
inline bool make_tmap_halves(CUtensorMap* map, void* data, bool half, long long rows) {
  const PFN_encodeTiled encode = get_encode_tiled();
  if (!encode) return false;
  const cuuint64_t dims[3] = {64, (cuuint64_t)rows, D / 64}, strides[2] = {D * 2, 128};
  const cuuint32_t box[3] = {64, TILE, D / 64}, steps[3] = {1, 1, 1};
  const auto make = [&] {
    return encode(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, data, dims, strides, box, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = make();
  if (rc == CUDA_ERROR_INVALID_CONTEXT) {      // the first CUDA work of this host thread
    cudaFree(nullptr);
    rc = make();
  }
  return rc == CUDA_SUCCESS;
}

// Floats of the attention's workspace: what blocks leave of the sequences that they share, and with weights the scores.
struct Workspace {
  long long partial, owners, lse2, scores, all;
  int ctas;
  bool cut;
};
inline int column_tiles_of_8(int columns) { return columns <= 8 ? 1 : columns <= 16 ? 2 : 4; }
inline Workspace workspace(long long rows, int kv_heads, int columns, int D, long long places, bool weighed) {
  Workspace w;
  const int nt = column_tiles_of_8(columns);
  const long long per = (long long)((columns + 8 * nt - 1) / (8 * nt)) * kv_heads;
  // sequences of up to 256 tokens are not cut: four tiles a warp take less than a join and what the cutting needs to know
  w.cut = places > 256;
  w.ctas = w.cut ? 148 * 2 : 0;
  w.partial = 0;
  w.owners = 2LL * w.ctas * 8 * nt * (D + 4);
  w.lse2 = w.owners + (w.cut ? (2 * rows * per + 3) / 4 * 4 : 0);
  w.scores = w.lse2 + (weighed ? (rows * kv_heads * columns + 3) / 4 * 4 : 0);
  w.all = w.scores + (weighed ? rows * kv_heads * places * columns : 0);
  return w;
}

template <typename T, int D, int NT>
int launch_attention(AttnArgs a, cudaStream_t st) {
  using Sh = Shape<D, NT>;
  static std::atomic<unsigned long long> allowed{0};       // devices on which the kernel may have its shared memory
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return launched(cudaErrorInvalidDevice);
  const unsigned long long bit = 1ull << (device & 63);
  constexpr int SMEM = Sh::SMEM;
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    const int rc = launched(cudaFuncSetAttribute(kv_attention_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (rc != 0) return rc;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  const int columns = a.S * a.group;
  const long long places = (long long)a.c.width << a.c.page_shift;
  const long long per = (columns + Sh::COLS - 1) / Sh::COLS * (long long)a.c.kv_heads, runs = a.c.rows * per;
  const long long room = (places + TILE - 1) / TILE, most = (START + (room > 1 ? room : 1)) * runs;
  if (runs > 0x7fffffffLL || per / a.c.kv_heads > 60000) return -2;
  const Workspace w = workspace(a.c.rows, a.c.kv_heads, columns, D, places, a.weights != nullptr);
  if (w.all > 0 && !a.partial) return -1;
  float* const space = a.partial;
  a.owners = reinterpret_cast<int2*>(space + w.owners);
  a.lse2 = a.weights ? space + w.lse2 : nullptr;
  a.scores = a.weights ? space + w.scores : nullptr;
  a.ctas = w.ctas;
  CUtensorMap map;
  if (!make_tmap_halves<D>(&map, a.c.data, std::is_same<T, __half>::value, ((long long)a.c.pages * 2 * a.c.kv_heads) << a.c.page_shift)) return -3;
  const long long grid = most < 148 * Sh::BLOCKS ? most : 148 * Sh::BLOCKS;
  int rc = launched(launch_after(kv_attention_kernel<T, D, NT>, dim3((unsigned)(w.cut || runs > grid ? grid : runs)), WARPS * 32, SMEM, st, 1,
                                 map, a));
  if (rc != 0) return rc;
  if (!a.weights) return w.cut ? launched(launch_after(kv_join_kernel<T, D, NT>, dim3((unsigned)runs), 256, 0, st, 1, a, (int)per)) : 0;
  const long long heads = (long long)a.c.rows * a.c.kv_heads;
  const int lanes = columns <= 4 ? 1 : 8, each = 256 / lanes;
  const long long most_chunks = (places + each - 1) / each, enough = (lanes == 1 ? 148 * 3 : 148 * 6) / heads + 1;
  const int chunks = (int)(most_chunks < 1 ? 1 : most_chunks < enough ? most_chunks : enough);
  const dim3 blocks((unsigned)heads, (unsigned)(chunks + (w.cut ? per / a.c.kv_heads : 0)));
  return launched(lanes == 1 ? launch_after(kv_weights_kernel<T, D, NT, 1>, blocks, 256, 0, st, 1, a, (int)per, chunks)
                             : launch_after(kv_weights_kernel<T, D, NT, 8>, blocks, 256, 0, st, 1, a, (int)per, chunks));
}

template <int D>
int launch_evict(const EvictArgs& a, cudaStream_t st) {
  const long long units = (long long)a.layers * a.c.rows * a.c.kv_heads, places = (long long)a.c.width << a.c.page_shift;
  if (a.budget >= places) return launched(launch_after(kv_lengths_kernel, dim3((unsigned)(a.c.rows + 255) / 256), 256, 0, st, 1, a));
  // few units: a cluster of large blocks for each, where its blocks have 2048 places each
  const bool few = units < 148;
  int blocks = 1;
  while (blocks < 8 && units * blocks * 2 <= 148 && places > 2048LL * blocks) blocks *= 2;
  // (16 clusters of 8 blocks are resident at once if two blocks fit on an SM, not with one: 15 then)
  constexpr int LARGEST = 16384, MOVE = 512, PER = 6, DEEP = 2, RING = MOVE * PER * DEEP * 16;
  const long long share = (places + blocks - 1) / blocks + 4;
  const int room = (int)(share < LARGEST ? share : LARGEST);
  static std::atomic<unsigned long long> allowed{0};       // devices on which the kernels may have their shared memory
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return launched(cudaErrorInvalidDevice);
  const unsigned long long bit = 1ull << (device & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    int rc = launched(cudaFuncSetAttribute(kv_select_kernel<512>, cudaFuncAttributeMaxDynamicSharedMemorySize, LARGEST * 4));
    if (rc == 0) rc = launched(cudaFuncSetAttribute(kv_select_kernel<1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, LARGEST * 4));
    if (rc == 0) rc = launched(cudaFuncSetAttribute(kv_move_cluster_kernel<D, MOVE, PER, DEEP>, cudaFuncAttributeMaxDynamicSharedMemorySize, RING));
    if (rc != 0) return rc;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  int members = 1;
  while (few && members < 8 && units * 2 * members * 2 <= 148) members *= 2;
  if (units * 2 * members > 0x7fffffffLL) return -2;
  const dim3 grid((unsigned)(units * blocks)), movers((unsigned)(units * 2 * members));
  const int rc = launched(few ? launch_after(kv_select_kernel<1024>, grid, 1024, room * 4, st, blocks, a, room)
                              : launch_after(kv_select_kernel<512>, grid, 512, room * 4, st, blocks, a, room));
  if (rc != 0) return rc;
  return launched(few ? launch_after(kv_move_cluster_kernel<D, MOVE, PER, DEEP>, movers, MOVE, RING, st, members, a)
                      : launch_after(kv_move_kernel<D, 256, 8>, movers, 256, 0, st, 1, a));
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
  return workspace(rows, kv_heads, heads / kv_heads * S, head_dim, places, weighed != 0).all;
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
  const int tiles = column_tiles_of_8(S * a.group);
#define ATTN(T, D)                                                                 \
  return tiles == 1   ? launch_attention<T, D, 1>(a, (cudaStream_t)stream)         \
         : tiles == 2 ? launch_attention<T, D, 2>(a, (cudaStream_t)stream)         \
                      : launch_attention<T, D, 4>(a, (cudaStream_t)stream)
  ATB_KV_TYPES(ATTN)
#undef ATTN
  return -1;
}

extern "C" int atb_kv_evict(void* data, const void* table, const void* lengths, void* weights, void* out, void* work, int layers,
                            int kv_heads, int head_dim, int page_shift, int pages, int rows, int width, long long table_stride,
                            long long places, int budget, int recent, void* stream, void* status) {
  if (rows <= 0) return 0;
  EvictArgs a;
  a.c = cache_of(data, table, table_stride, rows, width, pages, kv_heads, page_shift);
  a.lengths = (const int*)lengths;
  a.weights = (float*)weights;
  a.out = (int*)out;
  const long long units = (long long)layers * rows * kv_heads;
  a.first = (int*)work;
  a.source = a.first + units;
  a.kept = (float*)(a.source + units * budget);
  a.places = places;
  a.layer_elements = ((long long)pages * 2 * kv_heads << page_shift) * head_dim;
  a.budget = budget;
  a.recent = recent;
  a.layers = layers;
  a.status = (int*)status;
  if (head_dim == 64) return launch_evict<64>(a, (cudaStream_t)stream);
  if (head_dim == 128) return launch_evict<128>(a, (cudaStream_t)stream);
  return -1;
}
