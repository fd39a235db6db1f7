// Products with weights held in 4 bits: y[m, n] = sum_k x[m, k] (code[n, k] - 8) scale[n, k / G], for few rows m.
//
//   codes  uint8 [N][16 ceil(K / 32)]   byte i: column 2i low, column 2i + 1 high; filled up with 8s, which stand for 0
//   scales bf16  [N][ceil(K / G)]       G = 32, 64 or 128 columns share a scale
//
// Bound by the codes, N K / 2 bytes, for as many rows as a decode step has. The products run on the warp's matrix instruction
// (16 x 8 x 16) with 16 weight rows as its tall operand and 8 rows of x as the other. A code becomes code - 8 in the type of x
// by one AND-OR and one packed subtraction for two of them, exactly: 128 + code and 1024 + code are bf16 and fp16 numbers with
// the code in their last bits. The products with x are exact in fp32, sums of a group are fp32, and the scale, one per row and
// group, multiplies the sum of the group.
#include "common.cuh"

namespace {
using namespace atb;

constexpr int WARPS = 8;

template <typename T>
ATB_DEVICE void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && __is_same(T, __half))
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// codes at places p and p + 4 of a word, less 8, as two numbers of T
template <typename T>
ATB_DEVICE uint32_t weights_of(uint32_t w, int p) {
  if constexpr (__is_same(T, __half)) {
    const uint32_t u = ((w >> (4 * p)) & 0x000F000Fu) | 0x64006400u, eight = 0x64086408u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&eight));
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const uint32_t u = ((w >> (4 * p)) & 0x000F000Fu) | 0x43004300u, eight = 0x43084308u;
    const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&eight));
    return *reinterpret_cast<const uint32_t*>(&h);
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

// A block has 16 R rows of the weights and 8 NT rows of x; its warps take the groups in turn. A lane (r, q) reads the quarter q of
// a group of weight rows r and r + 8, V words (8 codes each), and of row r of x.
template <typename T, int V, int NT, int R>
__global__ void __launch_bounds__(WARPS * 32) w4_kernel(Args a) {
  constexpr int G = 32 * V;
  __shared__ float part[WARPS][16 * R][8 * NT + 1];
  grid_go();
  grid_wait();
  if (__syncthreads_or(threadIdx.x == 0 && *a.status != 0)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, q = lane & 3;
  const int n0 = blockIdx.x * 16 * R, m0 = blockIdx.y * 8 * NT;
  float acc[R][NT][4] = {};
  for (int g = warp; g < a.groups; g += WARPS) {
    uint32_t xf[NT][V][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int m = m0 + 8 * j + r;
      const T* row = reinterpret_cast<const T*>(a.x) + m * a.x_stride;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (m < a.M) u = load_x<T>(a, row, g * G + (q * V + v) * 8);
        xf[j][v][0] = __byte_perm(u.x, u.z, 0x5410);
        xf[j][v][1] = __byte_perm(u.x, u.z, 0x7632);
        xf[j][v][2] = __byte_perm(u.y, u.w, 0x5410);
        xf[j][v][3] = __byte_perm(u.y, u.w, 0x7632);
      }
    }
#pragma unroll
    for (int s = 0; s < R; ++s) {
      uint32_t w[2][V];
      float scale[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n = n0 + 16 * s + 8 * i + r, at = (g * 4 + q) * (4 * V);
        const bool in = n < a.N && at < a.row_bytes;
        const uint8_t* p = a.codes + (long long)n * a.row_bytes + at;
#pragma unroll
        for (int v = 0; v < V; ++v) w[i][v] = 0x88888888u;
        if (in) {
          if constexpr (V == 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            w[i][0] = u.x; w[i][1] = u.y; w[i][2] = u.z; w[i][3] = u.w;
          } else if constexpr (V == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            w[i][0] = u.x; w[i][1] = u.y;
          } else {
            w[i][0] = *reinterpret_cast<const uint32_t*>(p);
          }
        }
        scale[i] = n < a.N ? __bfloat162float(a.scales[(long long)n * a.groups + g]) : 0.f;
      }
      float d[NT][4] = {};
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int p = 0; p < 4; p += 2) {
          const uint32_t f[4] = {weights_of<T>(w[0][v], p), weights_of<T>(w[1][v], p), weights_of<T>(w[0][v], p + 1),
                                 weights_of<T>(w[1][v], p + 1)};
#pragma unroll
          for (int j = 0; j < NT; ++j) mma<T>(d[j], f, xf[j][v][p], xf[j][v][p + 1]);
        }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[s][j][e] = fmaf(scale[e >> 1], d[j][e], acc[s][j][e]);
    }
  }
#pragma unroll
  for (int s = 0; s < R; ++s)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[warp][16 * s + 8 * (e >> 1) + r][8 * j + 2 * q + (e & 1)] = acc[s][j][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * R * 8 * NT; i += WARPS * 32) {
    const int row = i % (16 * R), col = i / (16 * R), n = n0 + row, m = m0 + col;
    if (n >= a.N || m >= a.M) continue;
    float sum = a.bias ? to_f32<T>(reinterpret_cast<const T*>(a.bias)[n]) : 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) sum += part[k][row][col];
    reinterpret_cast<T*>(a.y)[(long long)m * a.N + n] = from_f32<T>(sum);
  }
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
int launch(const Args& a, cudaStream_t st) {
  const dim3 grid((a.N + 16 * R - 1) / (16 * R), (a.M + 8 * NT - 1) / (8 * NT));
  if (grid.y > 65535) return -2;
  return launch_after(w4_kernel<T, V, NT, R>, grid, WARPS * 32, 0, st, 1, a) == cudaSuccess ? 0 : -5;
}
template <typename T, int V>
int by_rows(const Args& a, cudaStream_t st) {
  if (a.M <= 8) return launch<T, V, 1, 1>(a, st);
  if (a.M <= 16) return launch<T, V, 2, 2>(a, st);
  return launch<T, V, 4, 2>(a, st);
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
               (K + group - 1) / group, x_stride, wide, (const int*)status};
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
  return rc == cudaSuccess ? 0 : -5;
}
