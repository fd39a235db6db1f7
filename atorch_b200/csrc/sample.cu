// The next token of every row of logits: temperature, top-k, top-p and min-p, drawn with given waiting times.
//
// w = exp((x - max) / T). The tokens in the order (larger logit, lower index) that are left are a prefix of it: the first `top_k`; of
// these the ones whose predecessors weigh less than top_p of what they weigh together; of these the ones with w >= min_p. Drawn is the
// token with the largest w / waiting time.
#include <cooperative_groups.h>
#include "row.cuh"

namespace {
using namespace atb;
namespace cg = cooperative_groups;

// Threads of a block; bins of a factor of 2 in weight, the last for all that is less; tokens that one block draws from; tokens that it
// puts in order by counting; parts of a step towards the end of the prefix where there are more
constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 20, ROOM = 4096, FEW = 256, SUB = 512;
constexpr double DOUBT = 1. / (1 << 24);         // of a row's weight: how near to a border sums in 32 bits are not trusted
constexpr float NOTHING = 1075.f;       // powers of two below the largest weight from which on a weight is 0 in 64 bits

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

ATB_DEVICE double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = (threadIdx.x & 31) < WARPS ? red[threadIdx.x & 31] : 0.;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}
// Sum over the threads before this one
template <typename N>
ATB_DEVICE N block_before(N v, N* red, N& all) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  N sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  __syncthreads();
  if (lane == 31) red[w] = sum;
  __syncthreads();
  const N x = lane < WARPS ? red[lane] : (N)0;
  N up = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N y = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += y;
  }
  all = __shfl_sync(0xffffffffu, up, 31);
  const N before = __shfl_sync(0xffffffffu, up - x, w);
  const N mine = __shfl_up_sync(0xffffffffu, sum, 1);
  return lane == 0 ? before : before + mine;
}

// Weights of a row: exactly, and in 32 bits as a power of two (how far below the largest) with what rounding the exponent left. Only logits
// above `least` have one: that is -inf, or, where the largest is +inf, every finite number.
struct Scale {
  float top, c, c_low, cap, least;       // c + c_low: log2(e) / T; distances are cut at `cap`
  double temp;
  ATB_DEVICE Scale(float top, double temp) : top(top), temp(temp) {
    const bool endless = top == INFINITY;
    const double d = endless ? 0. : fmin(1.4426950408889634 / temp, 1e38);
    c = (float)d;
    c_low = (float)(d - (double)c);
    cap = 1e36f / fmaxf(c, 1.f);
    least = endless ? 3.402823466e38f : -INFINITY;
  }
  ATB_DEVICE float below(float v) const { return fminf(top - v, cap); }            // (a NaN: cap)
  ATB_DEVICE float power(float v) const { return v > least ? below(v) * c : 1e30f; }
  ATB_DEVICE double exact(float v) const { return !(v > least) ? 0. : top == INFINITY ? 1. : exp(((double)v - (double)top) / temp); }
  // off by 2^-22 of itself at most (the special-function unit) and 2^-24 of the distance that rounding the logits' difference leaves
  ATB_DEVICE float weight(float v, float y) const {
    const float d = below(v), rest = fmaf(d, c_low, fmaf(d, c, -y)), w = fast_exp2(-y);
    return fmaf(w, -0.69314718f * rest, w);
  }
};

// What the blocks of a cluster read from each other
struct Shared {
  float top;
  int first;                                     // lowest index of the largest logit, for a temperature of 0
  double sum;                                    // of the weights that this block has
  double above, inside;                          // of those above the bin at hand, and in it
  unsigned long long low, high, least_above;     // keys of the bin at hand, and the least above it
  unsigned count[BINS], weight[BINS];            // tokens of a bin, their weights in units of 2^-14 of the bin's largest
  int listed, few_listed;
  double margin;                                 // how near the target comes to where the prefix might end otherwise
  unsigned long long few[FEW], cut;
  unsigned long long best_score;                 // fp64 bits
  int best_at;
};

// A row's tokens are shared by the blocks of a cluster, a block's by its threads, which keep P pieces in registers.
//
// Without filters every block draws from its share, relative to its own largest logit. With top-k or top-p the end of the prefix is looked
// for first: in a histogram of tokens and weights over the powers of two below the largest weight, where every thread has bins of its own.
// If no more than ROOM tokens lie in the bins down to the one where the prefix ends, the first block lists them, finds the end, and
// draws; if that bin alone has no more, it lists the bin, finds the end, and every block draws from its share; if there are more, all
// blocks look for the end together. Looking for the end: a few tokens are put in order and added up in 64 bits; of more, the keys' range is
// divided into SUB parts, and the part with the end again. Weights that several threads add up are whole numbers (2^-46 of the
// largest of the range), others are summed in one order, so the result does not depend on which thread comes first. Sums of
// thousands of weights in 32 bits are off by some 2^-26; where that might decide where the prefix ends, they are formed again in 64
// bits. A draw is decided in 64 bits: 32-bit arrival times only say which tokens have to be looked at.
template <typename T, int P>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(Args a) {
  // [BINS][THREADS]: weights in the low 22 bits, tokens above; then the list of keys, and behind it [4][SUB]: tokens of a part, its
  // weights in three limbs of 16 bits
  extern __shared__ __align__(16) unsigned own_bins[];
  unsigned long long* const list = reinterpret_cast<unsigned long long*>(own_bins);
  unsigned* const parts = own_bins + 2 * ROOM;
  static_assert(ROOM * 8 + 4 * SUB * 4 <= BINS * THREADS * 4, "they lie in the place of the bins");
  __shared__ Shared sh;
  __shared__ double red_d[32];
  __shared__ int red_i[32];
  __shared__ float red_f[33];
  cg::cluster_group cluster = cg::this_cluster();
  grid_go();
  grid_wait();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31;
  const bool leader = rank == 0;
  const long long row = blockIdx.x / blocks;
  const T* const x = (const T*)a.logits + row * a.stride;
  const float* const wait = a.waiting + row * a.wait_stride;
  const int part = ((a.V + blocks - 1) / blocks + 7) / 8 * 8, from = min(a.V, rank * part), to = min(a.V, from + part);
  constexpr int N = Piece<T>::N;
  const RowShare<T, P, THREADS> share(x, from, to, (reinterpret_cast<uintptr_t>(x) & 15) == 0);
  auto each = [&](auto f) {                      // f(logit, index)
    share.each([&](const Piece<T>& v, int i) {
#pragma unroll
                 for (int e = 0; e < N; ++e) f(v[e], i + e);
               }, f);
  };
  auto again = [&](auto f) {                     // the same from memory, for what happens seldom
    const int pieces = (reinterpret_cast<uintptr_t>(x) & 15) == 0 ? (to - from) / N : 0;
#pragma unroll 1
    for (int k = threadIdx.x; k < pieces; k += THREADS) {
      const Piece<T> v{reinterpret_cast<const uint4*>(x + from)[k]};
#pragma unroll
      for (int e = 0; e < N; ++e) f(v[e], from + k * N + e);
    }
#pragma unroll 1
    for (int i = from + pieces * N + threadIdx.x; i < to; i += THREADS) f(to_f32<T>(x[i]), i);
  };
  const double temp = a.t_rows ? a.t_rows[row] : a.t, p = a.p_rows ? a.p_rows[row] : a.p;
  double m = a.m_rows ? a.m_rows[row] : a.m;
  if (m > 1.) m = 1.;
  int k = a.k_rows ? a.k_rows[row] : a.k;
  if (k < 0 || k >= a.V) k = 0;
  const bool failed = *a.status != 0, by_weight = p < 1., unfiltered = k == 0 && !by_weight && !(m > 0.) && temp > 0.;
  if (unfiltered)                                // every waiting time is read: on their way to L2 under the look for the largest logit
    for (int i = from + (int)threadIdx.x * 32; i < to; i += THREADS * 32)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(__cvta_generic_to_global(wait + i)));
  auto answer = [&](int token, double logprob) {
    a.tokens[row] = failed ? 0 : token;
    a.logprobs[row] = failed ? -INFINITY : (float)logprob;
  };
  auto block_min = [&](int v) {
    v = __reduce_min_sync(0xffffffffu, v);
    __syncthreads();
    if (lane == 0) red_i[threadIdx.x >> 5] = v;
    __syncthreads();
    return __reduce_min_sync(0xffffffffu, red_i[lane & (WARPS - 1)]);
  };
  // a number of every block, added up in their order
  auto over_blocks = [&](double Shared::*which) {
    const double mine = lane < blocks ? cluster.map_shared_rank(&sh, lane)->*which : 0.;
    double sum = 0.;
    for (int i = 0; i < blocks; ++i) sum += __shfl_sync(0xffffffffu, mine, i);
    return sum;
  };

  // the largest logit: the block's, and without filters only that
  float top = -INFINITY;
  share.each([&](const Piece<T>& v, int) { top = fmaxf(top, v.top()); }, [&](float v, int) { top = fmaxf(top, v); });
  top = block_max(top, red_f);
  if (threadIdx.x == 0) {
    sh.top = top;
    sh.first = a.V;
    sh.listed = 0;
    sh.best_score = 0;
    sh.best_at = a.V;
  }
  auto row_top = [&] {
    return warp_max(lane < blocks ? cluster.map_shared_rank(&sh, lane)->top : -INFINITY);
  };
  if (!unfiltered) {
    cluster.sync();
    top = row_top();
    if (top == -INFINITY || !(temp > 0.)) {
      int first = a.V;
      if (top > -INFINITY) again([&](float v, int i) { if (v == top) first = min(first, i); });
      first = __reduce_min_sync(0xffffffffu, first);
      if (lane == 0) atomicMin(&sh.first, first);
      cluster.sync();
      if (leader && threadIdx.x == 0) {
        for (int i = 0; i < blocks; ++i) first = min(first, cluster.map_shared_rank(&sh, i)->first);
        if (top == -INFINITY) answer(0, -INFINITY);
        else answer(first, 0.);
      }
      cluster.sync();
      return;
    }
  } else {
    __syncthreads();
  }
  const Scale scale(top, temp);

  // The block's tokens that f(append) calls append(key) with as often as the thread says it will, in the list; behind it those of the other
  // blocks in the first one's. Returns how many there are there.
  auto gather = [&](int mine, auto f) {
    int all, at = block_before(mine, red_i, all);
    if (threadIdx.x == 0) sh.listed = all;
    f([&](unsigned long long key) {
      if (at < ROOM) list[at] = key;
      ++at;
    });
    cluster.sync();
    if (!leader) return 0;
    const int listed = lane < blocks ? cluster.map_shared_rank(&sh, lane)->listed : 0;
    int before = 0, n = 0;
    for (int i = 0; i < blocks; ++i) {
      const int u = __shfl_sync(0xffffffffu, listed, i);
      if (i < (int)threadIdx.x >> 5) before += u;
      n += u;
    }
    const int r = threadIdx.x >> 5;              // a warp for each of the others
    if (r > 0 && r < blocks) {
      const unsigned long long* const other = cluster.map_shared_rank(list, r);
      const int more = __shfl_sync(0xffffffffu, listed, r);
#pragma unroll 4
      for (int i = lane; i < more; i += 32)
        if (before + i < ROOM) list[before + i] = other[i];
    }
    __syncthreads();
    return min(n, ROOM);
  };
  // keys of the first n of them in their order, by counting those before each (n <= FEW): of this thread's place
  auto put_in_order = [&](const unsigned long long* from, int n) {
    const unsigned long long key = (int)threadIdx.x < n ? from[threadIdx.x] : 0;
    int place = n;
    if ((int)threadIdx.x < n) {
      place = 0;
#pragma unroll 8
      for (int i = 0; i < n; ++i) place += from[i] > key;
    }
    __syncthreads();
    if ((int)threadIdx.x < n) sh.few[place] = key;
    __syncthreads();
    return (int)threadIdx.x < n ? sh.few[threadIdx.x] : 0ull;
  };

  // The end of the prefix among the keys that `keys(f)` calls f(key) with, those in [low, high], n of them at most: the least key whose
  // predecessors are fewer than `target` tokens (by count), or weigh less. `before` come in front of them. With LOCAL the first block alone has them all.
  double margin = 0.;
  auto end_of_prefix = [&](auto local, auto keys, unsigned long long low, unsigned long long high, int n, bool count, double target, double before) {
    constexpr bool LOCAL = decltype(local)::value;
    const int members = LOCAL ? 1 : blocks;
    auto meet = [&] {
      if constexpr (LOCAL) __syncthreads();
      else cluster.sync();
    };
    auto of = [&](int i) -> Shared* {
      if constexpr (LOCAL) return &sh;
      else return cluster.map_shared_rank(&sh, i);
    };
    while (n > FEW && low != high) {
      const int shift = max(0, 64 - __clzll(high - low) - 9);      // SUB parts at most
      const int up = 46 + min((int)scale.power(value_of(high)), 900);
      const double unit = ldexp(1., -up), per = ldexp(1., up);
      for (int i = threadIdx.x; i < 4 * SUB; i += THREADS) parts[i] = 0;
      __syncthreads();
      keys([&](unsigned long long key) {
        if (key < low || key > high) return;
        const int s = (int)((high - key) >> shift);
        atomicAdd(parts + s, 1u);
        if (count) return;
        const unsigned long long q = (unsigned long long)(scale.exact(value_of(key)) * per);
        atomicAdd(parts + 1 * SUB + s, (unsigned)q & 0xffffu);
        atomicAdd(parts + 2 * SUB + s, (unsigned)(q >> 16) & 0xffffu);
        atomicAdd(parts + 3 * SUB + s, (unsigned)(q >> 32));
      });
      meet();
      static_assert(SUB == THREADS, "a thread has one part");
      unsigned mine_n = 0;
      unsigned long long mine_w = 0;
      for (int i = 0; i < members; ++i) {
        const unsigned* s = parts;
        if constexpr (!LOCAL) s = cluster.map_shared_rank(parts, i);
        mine_n += s[threadIdx.x];
        if (!count)
          mine_w += s[SUB + threadIdx.x] + ((unsigned long long)s[2 * SUB + threadIdx.x] << 16) + ((unsigned long long)s[3 * SUB + threadIdx.x] << 32);
      }
      double all;
      const double mine = count ? (double)mine_n : (double)mine_w * unit, till = block_before(mine, red_d, all) + before;
      // the first part at whose end the target is reached, or the last that has tokens
      int hit = block_min(mine_n > 0 && till + mine >= target ? (int)threadIdx.x : SUB);
      if (hit == SUB) hit = -block_min(mine_n > 0 ? -(int)threadIdx.x : 1);
      __syncthreads();
      if ((int)threadIdx.x == hit) {
        red_d[0] = till;
        red_i[0] = (int)mine_n;
      }
      meet();                                    // (the parts have been read by all)
      before = red_d[0];
      n = red_i[0];
      const unsigned long long top_key = high - ((unsigned long long)max(hit, 0) << shift), width = (1ull << shift) - 1;
      low = top_key - low > width ? top_key - width : low;
      high = top_key;
      __syncthreads();
    }
    // few: in their order
    if (threadIdx.x == 0) sh.few_listed = 0;
    __syncthreads();
    keys([&](unsigned long long key) {
      if (key < low || key > high) return;
      const int at = atomicAdd(&sh.few_listed, 1);
      if (at < FEW) sh.few[at] = key;
    });
    meet();
    if (leader) {
      n = min(sh.few_listed, FEW);
      for (int r = 1; r < members; ++r) {
        const Shared* s = of(r);
        const int more = s->few_listed;
        __syncthreads();
        for (int i = threadIdx.x; i < more && n + i < FEW; i += THREADS) sh.few[n + i] = s->few[i];
        n = min(n + more, FEW);
      }
      __syncthreads();
      const unsigned long long key = put_in_order(sh.few, n);
      double all;
      const double w = (int)threadIdx.x >= n ? 0. : count ? 1. : scale.exact(value_of(key));
      const double till = block_before(w, red_d, all) + before;
      const int left = block_min((int)threadIdx.x < n && till >= target ? (int)threadIdx.x : n);
      if (threadIdx.x == 0) {
        sh.cut = sh.few[max(left, 1) - 1];
        sh.margin = INFINITY;
      }
      __syncthreads();
      // (distances as the bits of numbers that are not negative)
      if ((int)threadIdx.x < n && ((int)threadIdx.x == left || (int)threadIdx.x == left - 1))
        atomicMin(reinterpret_cast<unsigned long long*>(&sh.margin),
                  (unsigned long long)__double_as_longlong(fmin(fabs(till - target), fabs(till + w - target))));
    }
    meet();
    const unsigned long long end = of(0)->cut;
    margin = of(0)->margin;
    meet();
    return end;
  };
  // keys of which no token so many powers of two below the largest has a greater one, or a lesser one
  auto highest_at = [&](float y) { return key_of(scale.c > 0.f ? scale.top - y / scale.c * 0.99999f : scale.top, 0); };
  auto lowest_at = [&](float y) { return scale.c > 0.f ? key_of(scale.top - y / scale.c * 1.00001f, 0xffffffffu) : 0ull; };
  // the weight of the whole row in 64 bits, by the first block
  auto exact_total = [&] {
    double w = 0.;
#pragma unroll 4
    for (int i = threadIdx.x; i < a.V; i += THREADS) w += scale.exact(to_f32<T>(x[i]));
    return block_sum(w, red_d);
  };
  // of the block's threads' tokens the one with the largest score, the lowest of equal ones
  auto best_of_block = [&](double score, int token) {
    if (score >= 0.) atomicMax(&sh.best_score, (unsigned long long)__double_as_longlong(score));
    __syncthreads();
    if (score >= 0. && (unsigned long long)__double_as_longlong(score) == sh.best_score) atomicMin(&sh.best_at, token);
  };
  auto score_of = [&](double w, float t) { return t >= 0.f ? w / (double)t : 0.; };

  unsigned long long cut = 0;                    // tokens with keys of at least this are left
  if (k > 0 || by_weight) {
    // one look at the row: tokens and weights of the bins, and all weights; a token without weight does not count
#pragma unroll
    for (int i = 0; i < BINS; ++i) own_bins[i * THREADS + threadIdx.x] = 0;
    float sum = 0.f;
    each([&](float v, int) {
      const float y = scale.power(v);
      if (!(y < NOTHING)) return;
      const int bin = min((int)y, BINS - 1);
      const float w = scale.weight(v, y);
      sum += w;
      // (w 2^bin lies in (1/2, 1], in the last bin below; 1.5 2^(23 - 14): adding it leaves the nearest unit in the low bits)
      const unsigned q = __float_as_uint(w * __int_as_float((127 + bin) << 23) + 768.f) - __float_as_uint(768.f);
      own_bins[bin * THREADS + threadIdx.x] += (1u << 22) + q;
    });
    const double total_own = block_sum(sum, red_d);
    if (threadIdx.x == 0) sh.sum = total_own;
    for (int bin = threadIdx.x >> 5; bin < BINS; bin += WARPS) {
      unsigned n = 0, w = 0;
#pragma unroll
      for (int i = 0; i < THREADS; i += 32) {
        const unsigned u = own_bins[bin * THREADS + i + lane];
        n += u >> 22;
        w += u & ((1u << 22) - 1);
      }
      n = __reduce_add_sync(0xffffffffu, n);
      w = __reduce_add_sync(0xffffffffu, w);
      if (lane == 0) {
        sh.count[bin] = n;
        sh.weight[bin] = w;
      }
    }
    cluster.sync();
    double total = over_blocks(&Shared::sum), w_to = 0.;      // tokens and weights down to the lane's bin
    unsigned n_to = 0;
    if (lane < BINS) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < blocks) {
          const Shared* s = cluster.map_shared_rank(&sh, i);
          n_to += s->count[lane];
          w_to += s->weight[lane];
        }
    }
    w_to *= (double)__int_as_float((127 - 14 - lane) << 23);
    const unsigned n_bin = n_to;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, n_to, o);
      const double d = __shfl_up_sync(0xffffffffu, w_to, o);
      if (lane >= o) {
        n_to += u;
        w_to += d;
      }
    }
    const unsigned counted = __shfl_sync(0xffffffffu, n_to, BINS - 1);
    const bool by_count = k > 0 && (unsigned)k < counted;       // (fewer have weight: top_k leaves them all)
    int bin = BINS - 1;                          // the prefix ends in this bin or before
    if (by_count) {
      bin = __ffs(__ballot_sync(0xffffffffu, lane < BINS && n_to >= (unsigned)k)) - 1;
    } else if (by_weight) {
      // (the bins' weights are rounded: a bin more rather than one too few)
      const unsigned hit = __ballot_sync(0xffffffffu, lane < BINS - 1 && w_to >= p * total * 1.0002);
      bin = hit ? __ffs(hit) - 1 : BINS - 1;
    }

    if (__shfl_sync(0xffffffffu, n_to, bin) <= ROOM) {
      const float until = bin == BINS - 1 ? NOTHING : (float)(bin + 1);
      int mine = 0;
      for (int i = 0; i <= bin; ++i) mine += own_bins[i * THREADS + threadIdx.x] >> 22;
      const int n = gather(mine, [&](auto append) { each([&](float v, int i) { if (scale.power(v) < until) append(key_of(v, i)); }); });
      if (leader) {
        double all = 0., score = -1.;
        int token = a.V;
        if (n <= FEW) {
          // in their order, all filters at once
          const unsigned long long key = put_in_order(list, n);
          const int j = threadIdx.x;
          const double w = j < n ? scale.exact(value_of(key)) : 0.;
          const float t = j < n ? wait[index_of(key)] : 0.f;
          const double before = block_before(by_count && j >= k ? 0. : w, red_d, all);
          int left;
          for (int round = 0;; ++round) {
            const double target = by_weight ? p * (by_count ? all : total) : INFINITY;
            const bool behind = j > 0 && (before >= target || w < m);
            left = block_min(j >= n || (by_count && j >= k) || behind ? j : THREADS);
            if (!by_weight || by_count || round > 0 || !__syncthreads_or(j <= left && fabs(before - target) < DOUBT * total)) break;
            total = exact_total();
          }
          all = block_sum(j < left ? w : 0., red_d);
          if (j < left && w > 0.) {
            score = score_of(w, t);
            token = (int)index_of(key);
          }
        } else {
          auto keys = [&](auto f) {
#pragma unroll 4
            for (int i = threadIdx.x; i < n; i += THREADS) f(list[i]);
          };
          const unsigned long long high = highest_at(0.f), low = lowest_at(until);
          if (by_count) cut = end_of_prefix(std::true_type(), keys, low, high, n, true, (double)k, 0.);
          if (by_weight) {
            if (by_count) {
              double w = 0.;
              keys([&](unsigned long long key) { if (key >= cut) w += scale.exact(value_of(key)); });
              total = block_sum(w, red_d);
            }
            const unsigned long long from_key = max(low, cut);
            unsigned long long end = end_of_prefix(std::true_type(), keys, from_key, high, n, false, p * total, 0.);
            if (!by_count && margin < DOUBT * total) {
              total = exact_total();
              end = end_of_prefix(std::true_type(), keys, from_key, high, n, false, p * total, 0.);
            }
            cut = max(cut, end);
          }
          constexpr int EACH = ROOM / THREADS;
          float t[EACH];
#pragma unroll
          for (int e = 0; e < EACH; ++e) {
            const int j = threadIdx.x + e * THREADS;
            t[e] = j < n && list[j] >= cut ? wait[index_of(list[j])] : -1.f;
          }
#pragma unroll
          for (int e = 0; e < EACH; ++e) {
            const int j = threadIdx.x + e * THREADS;
            if (j >= n || list[j] < cut) continue;
            const double w = scale.exact(value_of(list[j]));
            if (w < m || w == 0.) continue;
            all += w;
            const double s = score_of(w, t[e]);
            const int i = (int)index_of(list[j]);
            if (s > score || (s == score && i < token)) {
              score = s;
              token = i;
            }
          }
          all = block_sum(all, red_d);
        }
        best_of_block(score, token);
        __syncthreads();
        if (threadIdx.x == 0) {
          const int i = sh.best_at;
          answer(i, log(scale.exact(to_f32<T>(x[i])) / all));
        }
      }
      cluster.sync();                            // the first has read the others' lists
      return;
    }

    // Too many to draw from for one block, but not those of the bin where the prefix ends: one block finds the end.
    int at_bin = bin;
    if (!by_count) {
      const unsigned hit = __ballot_sync(0xffffffffu, lane < BINS - 1 && w_to >= p * total);
      at_bin = min(bin, hit ? __ffs(hit) - 1 : BINS - 1);
    }
    bool found = false;
    if (__shfl_sync(0xffffffffu, n_bin, at_bin) <= ROOM && !(by_count && by_weight)) {
      const double target = by_count ? (double)k : p * total;
      float w_above = 0.f, w_inside = 0.f;
      const int mine = own_bins[at_bin * THREADS + threadIdx.x] >> 22;
      const int n = gather(mine, [&](auto append) {
        each([&](float v, int i) {
          const float y = scale.power(v);
          if (!(y < NOTHING)) return;
          const int b = min((int)y, BINS - 1);
          if (b > at_bin) return;
          const float w = scale.weight(v, y);
          if (b < at_bin) w_above += w;
          else {
            w_inside += w;
            append(key_of(v, i));
          }
        });
        // (before the blocks meet)
        const double above = block_sum((double)w_above, red_d), inside = block_sum((double)w_inside, red_d);
        if (threadIdx.x == 0) {
          sh.above = above;
          sh.inside = inside;
        }
      });
      double before = by_count ? (double)(at_bin > 0 ? __shfl_sync(0xffffffffu, n_to, max(at_bin - 1, 0)) : 0u) : over_blocks(&Shared::above);
      const double inside = over_blocks(&Shared::inside);
      found = by_count || (target > before * (1. + DOUBT) && target < (before + inside) * (1. - DOUBT));      // (its weights are rounded)
      if (found) {
        if (leader) {
          auto keys = [&](auto f) {
#pragma unroll 4
            for (int i = threadIdx.x; i < n; i += THREADS) f(list[i]);
          };
          end_of_prefix(std::true_type(), keys, lowest_at(at_bin == BINS - 1 ? NOTHING : (float)(at_bin + 1)), highest_at((float)at_bin), n, by_count, target, before);
        }
        cluster.sync();
        cut = cluster.map_shared_rank(&sh, 0)->cut;
        found = by_count || cluster.map_shared_rank(&sh, 0)->margin >= DOUBT * total;
      }
      cluster.sync();
    }

    // Too many in that bin, or too near to a border, or both selections, one after the other: all blocks look for the end.
    for (int which = by_count ? 0 : 1; which < (by_weight ? 2 : 1) && !found; ++which) {
      const bool count = which == 0;
      if (which == (by_count ? 0 : 1)) cut = 0;
      if (!count && by_count) {                  // of what top_k has left
        float s = 0.f;
        again([&](float v, int i) { if (key_of(v, i) >= cut) s += scale.weight(v, scale.power(v)); });
        const double own = block_sum(s, red_d);
        if (threadIdx.x == 0) sh.sum = own;
        cluster.sync();
        total = over_blocks(&Shared::sum);
      }
      const double target = count ? (double)k : p * total;
      at_bin = bin;
      if (!count) {
        const unsigned hit = __ballot_sync(0xffffffffu, lane < BINS - 1 && w_to >= target);
        at_bin = min(bin, hit ? __ffs(hit) - 1 : BINS - 1);
      }
      double before = 0.;
      unsigned long long low = 0, high = 0, least_above = ~0ull;
      unsigned inside = 0;
      int way = 0;                               // the bins' rounded weights may be a bin off: up or down from there
      while (true) {
        float w_above = 0.f, w_inside = 0.f;
        unsigned n_above = 0, n_inside = 0;
        unsigned long long lo = ~0ull, hi = 0, over = ~0ull;
        again([&](float v, int i) {
          const float y = scale.power(v);
          if (!(y < NOTHING)) return;
          const int b = min((int)y, BINS - 1);
          const unsigned long long key = key_of(v, i);
          if (b > at_bin || key < cut) return;
          const float w = scale.weight(v, y);
          if (b < at_bin) {
            w_above += w;
            ++n_above;
            over = min(over, key);
          } else {
            w_inside += w;
            ++n_inside;
            lo = min(lo, key);
            hi = max(hi, key);
          }
        });
        const double above_own = block_sum(count ? (double)n_above : (double)w_above, red_d), inside_own = block_sum((double)w_inside, red_d);
        if (threadIdx.x == 0) {
          sh.above = above_own;
          sh.inside = inside_own;
          sh.low = sh.least_above = ~0ull;
          sh.high = 0;
          sh.listed = 0;
        }
        __syncthreads();
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
          hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
          over = min(over, __shfl_xor_sync(0xffffffffu, over, o));
        }
        n_inside = __reduce_add_sync(0xffffffffu, n_inside);
        if (lane == 0) {
          atomicMin(&sh.low, lo);
          atomicMin(&sh.least_above, over);
          atomicMax(&sh.high, hi);
          atomicAdd(&sh.listed, (int)n_inside);
        }
        cluster.sync();
        const double in = over_blocks(&Shared::inside);
        before = over_blocks(&Shared::above);
        low = least_above = ~0ull;
        high = 0;
        inside = 0;
        for (int i = 0; i < blocks; ++i) {
          const Shared* s = cluster.map_shared_rank(&sh, i);
          inside += s->listed;
          low = min(low, s->low);
          high = max(high, s->high);
          least_above = min(least_above, s->least_above);
        }
        cluster.sync();
        if (count) break;
        if (target <= before && at_bin > 0 && way <= 0) {
          --at_bin;
          way = -1;
        } else if ((target > before + in || high == 0) && at_bin < bin && way >= 0) {
          ++at_bin;
          way = 1;
        } else {
          break;
        }
      }
      if (high == 0 || (target <= before && least_above != ~0ull)) {       // it ends with the bin above
        if (least_above != ~0ull) cut = max(cut, least_above);
        continue;
      }
      auto keys = [&](auto f) { again([&](float v, int i) { f(key_of(fmaxf(v, -INFINITY), i)); }); };
      unsigned long long end = end_of_prefix(std::false_type(), keys, max(low, cut), high, (int)inside, count, target, before);
      if (!count && margin < DOUBT * total) {
        double w_all = 0., w_above = 0.;
        again([&](float v, int i) {
          const unsigned long long key = key_of(fmaxf(v, -INFINITY), i);
          if (key < cut) return;
          const double w = scale.exact(v);
          w_all += w;
          if (key > high) w_above += w;
        });
        w_all = block_sum(w_all, red_d);
        w_above = block_sum(w_above, red_d);
        if (threadIdx.x == 0) {
          sh.sum = w_all;
          sh.above = w_above;
        }
        cluster.sync();
        total = over_blocks(&Shared::sum);
        before = over_blocks(&Shared::above);
        end = end_of_prefix(std::false_type(), keys, max(low, cut), high, (int)inside, count, p * total, before);
      }
      cut = max(cut, end);
    }
  }

  // The draw: the best arrival in 32 bits, how near the next best of the same thread comes, and the sum of what is left.
  float sum = 0.f, best = -INFINITY, next = -INFINITY;
  int at = -1;
  bool seen = false;
  auto arrival = [&](float y, float t) { return -y - __log2f(t); };        // (a NaN where t is negative or one: passed over)
  auto arrives = [&](float s, int i) {
    seen = true;
    next = fmaxf(next, fminf(best, s));
    at = s > best ? i : at;
    best = fmaxf(best, s);
  };
  const double most_below = m > 0. ? -temp * log(m) : INFINITY;       // distance from the largest logit
  const float surely = (float)most_below * (1.f - 1e-6f), never = (float)most_below * (1.f + 1e-6f);
  auto is_left = [&](float v, int i) {
    if (cut != 0 && key_of(v, i) < cut) return false;
    if (!(m > 0.)) return true;
    if (scale.top == INFINITY) return true;      // (all that have weight weigh 1)
    const float d = scale.below(v);
    return d <= surely || (d <= never && !(scale.exact(v) < m));
  };
  if (unfiltered) {
    auto one = [&](float v, float t, int i) {
      const float y = scale.power(v);
      sum += scale.weight(v, y);
      arrives(arrival(y, t), i);
    };
    const bool wide = (reinterpret_cast<uintptr_t>(wait) & 15) == 0;
    share.each([&](const Piece<T>& v, int i) {
                 float t[N];
                 if (wide) {
#pragma unroll
                   for (int e = 0; e < N; e += 4) {
                     const float4 u = *reinterpret_cast<const float4*>(wait + i + e);
                     t[e] = u.x; t[e + 1] = u.y; t[e + 2] = u.z; t[e + 3] = u.w;
                   }
                 } else {
#pragma unroll
                   for (int e = 0; e < N; ++e) t[e] = wait[i + e];
                 }
#pragma unroll
                 for (int e = 0; e < N; ++e) one(v[e], t[e], i + e);
               }, [&](float v, int i) { one(v, wait[i], i); });
  } else {
    auto one = [&](float v, float y, float t, int i) {
      sum += scale.weight(v, y);
      arrives(arrival(y, t), i);
    };
    share.each([&](const Piece<T>& v, int i) {
                 float y[N], t[N];
                 bool left[N];
#pragma unroll
                 for (int e = 0; e < N; ++e) {
                   y[e] = scale.power(v[e]);
                   left[e] = y[e] < NOTHING && is_left(v[e], i + e);
                   t[e] = left[e] ? wait[i + e] : 0.f;
                 }
#pragma unroll
                 for (int e = 0; e < N; ++e)
                   if (left[e]) one(v[e], y[e], t[e], i + e);
               }, [&](float v, int i) {
                 const float y = scale.power(v);
                 if (y < NOTHING && is_left(v, i)) one(v, y, wait[i], i);
               });
  }
  const double sum_own = block_sum((double)sum, red_d);
  const float block_best = block_max(best, red_f);
  if (threadIdx.x == 0) sh.sum = sum_own;
  // what may come first when it is looked at exactly
  const float near = block_best - 2e-5f * (2.f + fminf(fabsf(block_best), 1e30f));
  double score = -1.;
  int token = a.V;
  auto look = [&](float v, int i) {
    const double w = scale.exact(v);
    if (w == 0.) return;
    const double s = score_of(w, wait[i]);
    if (s > score || (s == score && i < token)) {
      score = s;
      token = i;
    }
  };
  if (at >= 0 && best >= near) {
    if (next >= near)
      again([&](float v, int i) {
        const float y = scale.power(v);
        if (y < NOTHING && is_left(v, i) && arrival(y, wait[i]) >= near) look(v, i);
      });
    else
      look(to_f32<T>(x[at]), at);
  }
  best_of_block(score, token);
  if (__syncthreads_or(seen) && sh.best_at == a.V) {
    // none: every waiting time is infinite, or a token without weight arrived at once
    again([&](float v, int i) { if (scale.power(v) < NOTHING && is_left(v, i)) look(v, i); });
    best_of_block(score, token);
  }
  cluster.sync();
  if (leader && threadIdx.x < 32) {
    // the blocks' tokens relative to the row's largest logit
    const Shared* s = cluster.map_shared_rank(&sh, lane < blocks ? lane : 0);
    const float own = lane < blocks ? s->top : -INFINITY;
    top = warp_max(own);
    const Scale all(top, temp);
    double w = lane < blocks && own > -INFINITY ? s->sum * (unfiltered ? all.exact(own) : 1.) : 0.;
    double sum = 0.;
    for (int i = 0; i < blocks; ++i) sum += __shfl_sync(0xffffffffu, w, i);
    int i = lane < blocks ? s->best_at : a.V;
    w = i < a.V ? all.exact(to_f32<T>(x[i])) : 0.;
    score = i < a.V && w > 0. ? score_of(w, wait[i]) : -1.;
    for (int o = 16; o > 0; o >>= 1) {
      const double other = __shfl_xor_sync(0xffffffffu, score, o), other_w = __shfl_xor_sync(0xffffffffu, w, o);
      const int other_i = __shfl_xor_sync(0xffffffffu, i, o);
      if (other > score || (other == score && other_i < i)) {
        score = other;
        w = other_w;
        i = other_i;
      }
    }
    if (lane == 0) {
      if (top == -INFINITY || i >= a.V) answer(0, -INFINITY);
      else answer(i, log(w / sum));
    }
  }
  cluster.sync();
}

template <typename T, int P>
int launch(const Args& a, int rows, int blocks, cudaStream_t st) {
  constexpr int SMEM = BINS * THREADS * 4;
  static_assert(SMEM <= 48 << 10, "more has to be asked for");
  return launched(launch_after(sample_kernel<T, P>, dim3((unsigned)(rows * blocks)), THREADS, SMEM, st, blocks, a));
}
template <typename T>
int launch(const Args& a, int rows, cudaStream_t st) {
  constexpr int N = THREADS * (16 / sizeof(T));      // tokens of a piece for every thread
  // blocks of a row: as long as the GPU holds all of them at once and they have a piece for every thread
  int blocks = 1;
  while (blocks < 8 && (long long)rows * blocks * 2 <= 148 * 3 && a.V > N * blocks) blocks *= 2;
  const int part = (a.V + blocks - 1) / blocks + 8;
  // a thread's bins have room for the weights of 255 tokens, a block's parts for those of 65536
  while (blocks < 8 && a.V > blocks * 128 * THREADS) blocks *= 2;
  if (a.V > 8 * 128 * THREADS) return -2;
  if ((long long)rows * blocks > 0x7fffffffLL) return -2;
  if (part <= N) return launch<T, 1>(a, rows, blocks, st);
  if (part <= 2 * N) return launch<T, 2>(a, rows, blocks, st);
  if (part <= 4 * N) return launch<T, 4>(a, rows, blocks, st);
  return launch<T, 0>(a, rows, blocks, st);
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
  if (dtype == 0) return launch<__nv_bfloat16>(a, rows, st);
  if (dtype == 1) return launch<__half>(a, rows, st);
  if (dtype == 2) return launch<float>(a, rows, st);
  return -1;
}
