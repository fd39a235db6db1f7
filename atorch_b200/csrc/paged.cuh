// Pages of a key/value cache, and the cutting of its sequences into equal runs of work: what the caches of kv.cu and kv4.cu share.
//
// Sequence b's token p lies in page table[b][p / page size], place p % page size.
#pragma once
#include "common.cuh"

namespace atb {

struct Paging {
  const int* table;
  long long table_stride;
  int rows, width;       // sequences, pages a sequence may have
  int pages, kv_heads, page_shift;
};

// Page of token p of sequence b, or -1 where the table or the sequence does not have it.
ATB_DEVICE int page_of(const Paging& c, int b, int p) {
  const int i = p >> c.page_shift;
  if (b < 0 || b >= c.rows || i >= c.width) return -1;
  const int page = c.table[b * c.table_stride + i];
  return page < 0 || page >= c.pages ? -1 : page;
}
ATB_DEVICE int seen_length(const Paging& c, const int* lengths, int b, int* status) {
  const int n = lengths[b], most = c.width << c.page_shift;
  if (n > most) atomicCAS(status, 0, (int)ATB_ERR_BAD_INDEX);
  return max(0, min(n, most));
}
ATB_DEVICE long long warp_sum_ll(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Plan {
  long long units;
  int ctas;              // blocks with a run: run k is [k units / ctas, (k + 1) units / ctas)
  ATB_DEVICE long long begin(long long k) const { return k * units / ctas; }
  ATB_DEVICE int owner(long long u) const { return (int)(((u + 1) * ctas - 1) / units); }
};

// The work is one row of units: the tiles of TILE tokens of a sequence, once per head and column tile (`per` of them), one sequence
// behind another; what a sequence costs beside its tiles counts as START units before the first. Every block takes an equal run of
// it, which it finds for itself from the lengths on the device.
template <int TILE, int START, int WARPS>
struct Runs {
  ATB_HOST_DEVICE static int tiles_of(int n) {      // an empty sequence has its zeros written
    const int t = (n + TILE - 1) / TILE;
    return t > 1 ? t : 1;
  }
  // A run has a unit for every warp where there are enough.
  ATB_DEVICE static Plan plan(const Paging& c, const int* lengths, int per, int ctas, int* status) {
    long long total = 0;
    for (int b = threadIdx.x & 31; b < c.rows; b += 32) total += START + tiles_of(seen_length(c, lengths, b, status));
    Plan p;
    p.units = warp_sum_ll(total) * per;
    p.ctas = (int)max(1LL, min((long long)ctas, p.units / WARPS));
    return p;
  }
  // Sequence of unit u, its length and its first unit. Computed by a whole warp.
  ATB_DEVICE static void find(const Paging& c, const int* lengths, int per, long long u, int& b, int& len, long long& first,
                              int* status) {
    const int lane = threadIdx.x & 31;
    long long before = 0;
    for (int b0 = 0; b0 < c.rows; b0 += 32) {
      const int n = b0 + lane < c.rows ? seen_length(c, lengths, b0 + lane, status) : 0;
      const long long mine = b0 + lane < c.rows ? (long long)(START + tiles_of(n)) * per : 0;
      long long sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, u < before + sum);
      if (hit) {
        const int src = __ffs(hit) - 1;
        b = b0 + src;
        len = __shfl_sync(0xffffffffu, n, src);
        first = before + __shfl_sync(0xffffffffu, sum - mine, src);
        return;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
};

// 8 elements of a row as fp32, and back
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

ATB_DEVICE uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

}  // namespace atb
