// Products with weights held in 4 bits: y[m, n] = sum_k x[m, k] (code[n, k] - 8) scale[n, k / G], for few rows m.
//
//   codes  uint8 [N][16 ceil(K / 32)]   byte i: column 2i low, column 2i + 1 high; filled up with 8s, which stand for 0
//   scales bf16  [N][ceil(K / G)]       G = 32, 64 or 128 columns share a scale
//
// Bound by the codes, N K / 2 bytes, for as many rows as a decode step has. The products run on the warp's matrix instruction
// (16 x 8 x 16, fp32 sums) with 16 weight rows as its tall operand and 8 rows of x as the other. Two codes become code - 8 in the
// type of x by one AND-OR and one packed operation, exactly: 128 + code is a bf16 number with the code in its last bits, 1024 +
// code and 1024 + 16 code are such fp16 numbers (the known way of building small integers into the mantissa of a power of two). Products
// are exact in fp32, sums are fp32, and the scale of a row and group multiplies the sum of the group.
// Measured: 16 x 4096 x 22016 (47 MB) 24.3 us, 21.3 with x and a part of the codes in L2; 1 x 11008 x 4096 (23 MB) 13.1 and 11.9.
// Latency bounds it: the warps (14 of an SM, 80 and 128 registers) use 33 % and 27 % of the issue slots, and wait for loads first, then
// for operations on one another; a block stages its x and scales before its first product, and its cluster meets for the sum. Persistent
// blocks with equal runs of (strip, group) for every warp took 35 and 12 us, a prefetch of whole rows into L2 nothing off.
#include <atomic>
#include <cooperative_groups.h>
#include "common.cuh"

namespace {
using namespace atb;
namespace cg = cooperative_groups;

constexpr int WARPS = 8, AHEAD = 3, BATCH = 4;      // groups of codes asked for ahead; loads of x on their way at once

template <typename T>
ATB_DEVICE void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __half))
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
ATB_DEVICE uint32_t bits(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
ATB_DEVICE uint32_t bits(__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t*>(&v); }
// (x & mask) | magic in one operation (left to itself the compiler makes two of them)
ATB_DEVICE uint32_t and_or(uint32_t x, uint32_t mask, uint32_t magic) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(magic));
  return y;
}
// The codes of a word less 8: pair p holds places p and p + 4.
template <typename T>
ATB_DEVICE void weights_of(uint32_t w, uint32_t (&f)[4]) {
  if constexpr (__is_same(T, __half)) {
    const uint32_t magic = 0x64006400u, eight = 0x64086408u, by16 = 0x2c002c00u, less72 = 0xd480d480u;      // 1024, 1032, 1 / 16, -72
    const uint32_t hi = w >> 8;
    const uint32_t u[4] = {and_or(w, 0x000F000Fu, magic), and_or(w, 0x00F000F0u, magic), and_or(hi, 0x000F000Fu, magic),
                           and_or(hi, 0x00F000F0u, magic)};
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const __half2 h = *reinterpret_cast<const __half2*>(&u[p]);
      f[p] = bits(p & 1 ? __hfma2(h, *reinterpret_cast<const __half2*>(&by16), *reinterpret_cast<const __half2*>(&less72))
                        : __hsub2(h, *reinterpret_cast<const __half2*>(&eight)));
    }
  } else {
    const uint32_t magic = 0x43004300u, eight = 0x43084308u;                                                // 128, 136
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t u = and_or(w >> (4 * p), 0x000F000Fu, magic);
      f[p] = bits(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&eight)));
    }
  }
}

struct Args {
  const void* x;
  const uint8_t* codes;
  const __nv_bfloat16* scales;
  const void* bias;
  void* y;
  int M, N, K, row_bytes, groups;
  long long x_stride;
  int wide;          // rows of x can be read in 16-byte pieces
  int round;         // groups of x that shared memory holds
  const int* status;
};

// 8 elements of a row of x, zeros behind its end
template <typename T>
ATB_DEVICE uint4 load_x(const Args& a, const T* row, int k) {
  if (a.wide && k + 8 <= a.K) return *reinterpret_cast<const uint4*>(row + k);
  uint4 u;
  T* h = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = k + i < a.K ? row[k + i] : from_f32<T>(0.f);
  return u;
}
template <int V, int R>
struct Codes {
  uint32_t w[2 * R][V];
};

// A block has 128 R rows of the weights, 16 R a warp, and 8 NT rows of x; the blocks of a cluster have equal shares of the groups
// and add up their sums through each other's shared memory, in their order. A lane (r, q) reads the quarter q of a group of weight
// rows r + 8 i, V words (8 codes each), AHEAD groups ahead. What a block needs of x goes through shared memory in rounds of `round`
// groups, in the order in which the lanes need it: [group][word][row of x][quarter] pieces of 16 bytes, places p and p + 4 paired.
template <typename T, int V, int NT, int R>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 ? 3 : 2) w4_kernel(Args a) {
  constexpr int G = 32 * V, MX = 8 * NT, ROWS = 16 * R * WARPS;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float sums[MX][ROWS + 4];
  grid_go();
  grid_wait();
  const bool failed = *a.status != 0;      // nothing is stored then; the blocks of a cluster stay together
  cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, q = lane & 3;
  const int n_block = blockIdx.x / split * ROWS, m0 = blockIdx.y * MX, rows = min(MX, a.M - m0);
  const int g_begin = (int)((long long)a.groups * rank / split), g_end = (int)((long long)a.groups * (rank + 1) / split);
  uint4* const xs = reinterpret_cast<uint4*>(smem);                                             // [round][V][rows][4]
  float* const ss = reinterpret_cast<float*>(smem + (size_t)a.round * V * rows * 4 * 16);       // [round][ROWS] scales

  const uint8_t* row[2 * R];
#pragma unroll
  for (int i = 0; i < 2 * R; ++i)
    row[i] = a.codes + (long long)min(n_block + warp * 16 * R + 8 * i + r, a.N - 1) * a.row_bytes + q * (4 * V);
  const int last_at = a.row_bytes - 4 * V - q * (4 * V);       // behind the row's end x is 0, and any codes will do
  auto load = [&](Codes<V, R>& c, int g) {
    if (g >= g_end) return;
    const int at = min(g * (16 * V), last_at);
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) {
      const uint8_t* p = row[i] + at;
      if constexpr (V == 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        c.w[i][0] = u.x; c.w[i][1] = u.y; c.w[i][2] = u.z; c.w[i][3] = u.w;
      } else if constexpr (V == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        c.w[i][0] = u.x; c.w[i][1] = u.y;
      } else {
        c.w[i][0] = *reinterpret_cast<const uint32_t*>(p);
      }
    }
  };
  Codes<V, R> next[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(next[i], g_begin + i);

  float acc[R][NT][4] = {};
  int col[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) col[j] = min(8 * j + r, rows - 1) * 4 + q;           // columns without a row are not kept
  for (int g0 = g_begin; g0 < g_end; g0 += a.round) {
    const int here = min(a.round, g_end - g0);
    if (g0 > g_begin) __syncthreads();
    {
      const int piece = threadIdx.x % (4 * V), pq = piece & 3, pv = piece >> 2;
      const int step_m = WARPS * 8 / V % rows, step_g = WARPS * 8 / V / rows;
      int m = threadIdx.x / (4 * V) % rows, g = threadIdx.x / (4 * V) / rows;
      while (g < here) {        // several loads are on their way before the first is stored
        uint4 u[BATCH];
        int at[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          at[i] = g < here ? ((g * V + pv) * rows + m) * 4 + pq : -1;
          if (g < here) u[i] = load_x<T>(a, reinterpret_cast<const T*>(a.x) + (m0 + m) * a.x_stride, (g0 + g) * G + (pq * V + pv) * 8);
          g += step_g;
          m += step_m;
          if (m >= rows) {
            m -= rows;
            ++g;
          }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
          if (at[i] >= 0)
            xs[at[i]] = make_uint4(__byte_perm(u[i].x, u[i].z, 0x5410), __byte_perm(u[i].x, u[i].z, 0x7632),
                                   __byte_perm(u[i].y, u[i].w, 0x5410), __byte_perm(u[i].y, u[i].w, 0x7632));
      }
    }
    for (int i0 = threadIdx.x; i0 < here * ROWS; i0 += BATCH * WARPS * 32) {
      __nv_bfloat16 v[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int k = min(i0 + i * WARPS * 32, here * ROWS - 1);
        v[i] = a.scales[(long long)min(n_block + k % ROWS, a.N - 1) * a.groups + g0 + k / ROWS];
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i)
        if (i0 + i * WARPS * 32 < here * ROWS) ss[i0 + i * WARPS * 32] = __bfloat162float(v[i]);
    }
    __syncthreads();
    const float* const sl = ss + warp * 16 * R + r;
    for (int gt = 0; gt < here; gt += AHEAD) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int g = gt + i;
        if (g >= here) break;
        float d[R][NT][4] = {};
#pragma unroll
        for (int v = 0; v < V; ++v) {
          uint4 u[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j) u[j] = xs[(g * V + v) * rows * 4 + col[j]];
#pragma unroll
          for (int k = 0; k < R; ++k) {
            uint32_t f0[4], f1[4];
            weights_of<T>(next[i].w[2 * k][v], f0);
            weights_of<T>(next[i].w[2 * k + 1][v], f1);
            const uint32_t fa[4] = {f0[0], f1[0], f0[1], f1[1]}, fb[4] = {f0[2], f1[2], f0[3], f1[3]};
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              mma<T>(d[k][j], fa, u[j].x, u[j].y);
              mma<T>(d[k][j], fb, u[j].z, u[j].w);
            }
          }
        }
        load(next[i], g0 + g + AHEAD);
#pragma unroll
        for (int k = 0; k < R; ++k) {
          const float s0 = sl[g * ROWS + 16 * k], s1 = sl[g * ROWS + 16 * k + 8];
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[k][j][e] = fmaf(e < 2 ? s0 : s1, d[k][j][e], acc[k][j][e]);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < R; ++k)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[8 * j + 2 * q + (e & 1)][(warp * R + k) * 16 + 8 * (e >> 1) + r] = acc[k][j][e];
  if (split > 1) cluster.sync();
  else __syncthreads();
  // the blocks of a cluster finish the rows in turns, by the warp
  for (int i = warp * split + rank; i < ROWS / 32 * rows; i += WARPS * split) {
    const int at = i % (ROWS / 32) * 32 + lane, m = i / (ROWS / 32), n = n_block + at;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < split) v[k] = split == 1 ? sums[m][at] : *cluster.map_shared_rank(&sums[m][at], k);
    float sum = v[0];
#pragma unroll
    for (int k = 1; k < 8; ++k)
      if (k < split) sum += v[k];
    if (n >= a.N || failed) continue;
    if (a.bias) sum += to_f32<T>(reinterpret_cast<const T*>(a.bias)[n]);
    reinterpret_cast<T*>(a.y)[(long long)(m0 + m) * a.N + n] = from_f32<T>(sum);
  }
  if (split > 1) cluster.sync();         // the others have read this block's sums
}

// The weights themselves, [N][K], for products of many rows: a thread turns a word of 8 codes into 16 bytes.
template <typename T>
__global__ void __launch_bounds__(256) w4_expand_kernel(const uint8_t* codes, const __nv_bfloat16* scales, T* w, int K,
                                                        int row_bytes, int groups, int G) {
  grid_go();
  grid_wait();
  const int k = (blockIdx.y * 256 + threadIdx.x) * 8;
  if (k >= K) return;
  const long long n = blockIdx.x;
  const uint32_t u = *reinterpret_cast<const uint32_t*>(codes + n * row_bytes + k / 2);
  const float s = __bfloat162float(scales[n * groups + k / G]);
  uint4 o;
  T* h = reinterpret_cast<T*>(&o);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = from_f32<T>((float)((int)((u >> (4 * i)) & 15u) - 8) * s);
  *reinterpret_cast<uint4*>(w + n * K + k) = o;
}

template <typename T, int V, int NT, int R>
int launch(Args a, cudaStream_t st) {
  constexpr int G = 32 * V, MX = 8 * NT, ROWS = 16 * R * WARPS, MOST = 56 * 1024;
  static std::atomic<unsigned long long> allowed{0};       // devices on which the kernel may have its shared memory
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return launched(cudaErrorInvalidDevice);
  const unsigned long long bit = 1ull << (device & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    const int rc = launched(cudaFuncSetAttribute(w4_kernel<T, V, NT, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST));
    if (rc != 0) return rc;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  const long long blocks = (a.N + ROWS - 1LL) / ROWS, chunks = (a.M + MX - 1LL) / MX;
  if (chunks > 65535) return -2;
  // as many shares of the groups as keep all blocks on the GPU at once, of four groups at least: less would be outweighed by its
  // start
  const long long room = 148 * (NT == 1 ? 3 : 2) / (blocks * chunks);
  const int most = a.groups / 4, split = room < 2 || most < 2 ? 1 : room < 8 && room < most ? (int)room : most < 8 ? most : 8;
  const int rows = a.M < MX ? a.M : MX, group_bytes = G * 2 * rows + 4 * ROWS;
  const int share = (a.groups + split - 1) / split;
  a.round = MOST / group_bytes < share ? MOST / group_bytes / AHEAD * AHEAD : share;       // codes are asked for in turns of AHEAD
  if (blocks * split > 0x7fffffffLL) return -2;
  return launched(launch_after(w4_kernel<T, V, NT, R>, dim3((unsigned)(blocks * split), (unsigned)chunks), WARPS * 32,
                      (size_t)a.round * group_bytes, st, split, a));
}
template <typename T, int V>
int by_rows(const Args& a, cudaStream_t st) {
  if (a.M <= 8) return launch<T, V, 1, 1>(a, st);
  if (a.M <= 16) return launch<T, V, 2, 2>(a, st);
  return launch<T, V, 4, 1>(a, st);
}
template <typename T>
int by_group(const Args& a, int group, cudaStream_t st) {
  if (group == 32) return by_rows<T, 1>(a, st);
  if (group == 64) return by_rows<T, 2>(a, st);
  if (group == 128) return by_rows<T, 4>(a, st);
  return -1;
}
}  // namespace

extern "C" int atb_w4_linear(const void* x, const void* codes, const void* scales, const void* bias, void* y, int M, int N, int K,
                             int group, long long x_stride, int wide, int dtype, void* stream, void* status) {
  if (M <= 0 || N <= 0) return 0;
  const Args a{x, (const uint8_t*)codes, (const __nv_bfloat16*)scales, bias, y, M, N, K, (K + 31) / 32 * 16,
               (K + group - 1) / group, x_stride, wide, 0, (const int*)status};
  if (dtype == 0) return by_group<__nv_bfloat16>(a, group, (cudaStream_t)stream);
  if (dtype == 1) return by_group<__half>(a, group, (cudaStream_t)stream);
  return -1;
}

extern "C" int atb_w4_expand(const void* codes, const void* scales, void* w, int N, int K, int group, int dtype, void* stream) {
  if (N <= 0 || K <= 0) return 0;
  if (K % 8) return -1;
  const dim3 grid(N, (K / 8 + 255) / 256);
  if (grid.y > 65535) return -2;
  const int bytes = (K + 31) / 32 * 16, groups = (K + group - 1) / group;
  cudaError_t rc = cudaErrorInvalidValue;
  if (dtype == 0)
    rc = launch_after(w4_expand_kernel<__nv_bfloat16>, grid, 256, 0, (cudaStream_t)stream, 1, (const uint8_t*)codes,
                      (const __nv_bfloat16*)scales, (__nv_bfloat16*)w, K, bytes, groups, group);
  return launched(rc);
}
