// A row of logits that the blocks of a cluster share: pieces of 16 bytes, a thread's part of them, the order of tokens as a number.
#pragma once
#include <type_traits>
#include "common.cuh"

namespace atb {

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

// 16 bytes of a row
template <typename T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  uint4 u;
  ATB_DEVICE float operator[](int i) const { return to_f32<T>(reinterpret_cast<const T*>(&u)[i]); }
  // the largest of the piece; NaNs are passed over. 16-bit values are compared two at a time as they are.
  ATB_DEVICE float top() const {
    if constexpr (sizeof(T) == 4) {
      return fmaxf(fmaxf((*this)[0], (*this)[1]), fmaxf((*this)[2], (*this)[3]));
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2* h = reinterpret_cast<const T2*>(&u);
      const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      return fmaxf(to_f32<T>(m.x), to_f32<T>(m.y));
    }
  }
};
// The elements [from, to) of a row that a thread has: `each` calls f(piece, index of its first) for those in 16-byte pieces, where the
// row allows it (`wide`: it begins on 16 bytes; `from` is a multiple of 8), and one(value, index) for the others.
// P pieces of a thread stay in registers, all asked for at once; P = 0: they are read (from the first-level cache) every time. Two
// and four pay (4 beams of 32000 tokens 12.9 -> 11.9 us with what follows); eight leave room for three blocks an SM and pay as long as
// there are no more (192 beams 17.5 -> 14.5 us; with two blocks an SM, in two turns, 22).
template <typename T, int P, int THREADS>
struct RowShare {
  static constexpr int N = Piece<T>::N;
  const T* row;
  int from, to, pieces;
  Piece<T> kept[P > 0 ? P : 1];
  ATB_DEVICE RowShare(const T* row, int from, int to, bool wide) : row(row), from(from), to(to), pieces(wide ? (to - from) / N : 0) {
#pragma unroll
    for (int k = 0; k < P; ++k)
      if ((int)threadIdx.x + k * THREADS < pieces)
        kept[k] = Piece<T>{reinterpret_cast<const uint4*>(row + from)[threadIdx.x + k * THREADS]};
  }
  template <typename F, typename G>
  ATB_DEVICE void each(F f, G one) const {
    if constexpr (P > 0) {
#pragma unroll
      for (int k = 0; k < P; ++k)
        if ((int)threadIdx.x + k * THREADS < pieces) f(kept[k], from + ((int)threadIdx.x + k * THREADS) * N);
    } else {
#pragma unroll 4
      for (int i = threadIdx.x; i < pieces; i += THREADS)
        f(Piece<T>{reinterpret_cast<const uint4*>(row + from)[i]}, from + i * N);
    }
    for (int i = from + pieces * N + threadIdx.x; i < to; i += THREADS) one(to_f32<T>(row[i]), i);
  }
};

}  // namespace atb
