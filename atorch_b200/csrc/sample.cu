// The next token of every row of logits: temperature, top-k, top-p and min-p, drawn with given waiting times.
//
// w = exp((x - max) / T). The tokens in the order (larger logit, lower index) that are left are a prefix of it: the first `top_k`; of
// these the ones whose predecessors weigh less than top_p of what they weigh together; of these the ones with w >= min_p. Drawn is the
// token with the largest w / waiting time.
#include <atomic>
#include <cooperative_groups.h>
#include "row.cuh"

namespace {
using namespace atb;
namespace cg = cooperative_groups;

// Threads of a block; bins of a factor of 2 in weight, the last for all that is less; tokens of a block's list; tokens that are put in order
// by counting; parts of a step towards the end of the prefix where there are more
constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 20, ROOM = 4096, FEW = 256, SUB = 512;
constexpr float NOTHING = 1000.f;       // powers of two below the largest weight from which on a token has none

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

// (one copy of its code: a block runs most of its code once, and waits for it)
__device__ __noinline__ double exp_of(double x) { return exp(x); }
__device__ __noinline__ double quotient_of(double a, double b) { return a / b; }

// Weights of a row, relative to that of the largest logit. Only logits above `least` have one: that is -inf, or, where the largest is
// +inf, every finite number.
struct Scale {
  float top, c, c_rest, cap, least;      // c + c_rest: log2(e) / T; distances are cut at `cap`
  const double* powers;                  // 2^(-j / 32), in shared memory
  double per_temp;
  ATB_DEVICE Scale(float top, double temp, const double* powers) : top(top), powers(powers), per_temp(1. / temp) {
    const bool endless = top == INFINITY;
    const double c64 = endless ? 0. : fmin(1.4426950408889634 / temp, 1e38);
    c = (float)c64;
    c_rest = (float)(c64 - (double)c);
    cap = fminf(3.402823466e38f, 1e36f / c);
    least = endless ? 3.402823466e38f : -INFINITY;
  }
  ATB_DEVICE float below(float v) const { return fminf(top - v, cap); }            // (a NaN: cap)
  // how many powers of two below the largest weight
  ATB_DEVICE float power(float v) const { return v > least ? below(v) * c : 1e30f; }
  // The weight of a logit whose power is y < NOTHING, off by 2^-22 of itself at most (the special-function unit).
  ATB_DEVICE float rough(float v, float y) const {
    const float d = below(v), rest = fmaf(d, c_rest, fmaf(d, c, -y)), w = fast_exp2(-y);
    return fmaf(w, -0.69314718f * rest, w);
  }
  // The same off by 2^-30: 2^-y = 2^(-n / 32) 2^-r with n / 32 the nearest to y; the rest, with what the difference and the product were
  // rounded by, is in 32 bits off by 2^-30, and 2^-r - 1 four terms of its series, below 0.011. Where a prefix ends is decided by these: a
  // token at the end of one of thousands weighs 1e-5 of it, and a total of rough weights added up in 32 bits, off by 5e-8, moved the end
  // in one or two rows of a thousand. (All tokens' weights in 64 bits took 10 us for the look at 192 rows of 32000, these 8, the rough
  // ones 4.)
  template <typename T>
  ATB_DEVICE double weight(float v, float y) const {
    const float d = below(v);
    float rest = fmaf(d, c_rest, fmaf(d, c, -y));
    if constexpr (sizeof(T) == 4) {              // (16-bit logits have an exact difference, but for the tiniest)
      const float back = d - top;
      rest = d < cap ? fmaf((top - (d - back)) - (v + back), c, rest) : rest;
    }
    const float shifted = fmaf(y, 32.f, 12582912.f);      // 1.5 * 2^23: adding it leaves the nearest whole number in the low bits
    const int n = __float_as_int(shifted) - 0x4b400000;
    const float r = fmaf(shifted - 12582912.f, -1.f / 32.f, y) + rest;
    const float q = r * fmaf(r, fmaf(r, fmaf(r, 0.00961813f, -0.05550411f), 0.24022651f), -0.69314718f);      // (-ln 2)^k / k!
    const double w0 = powers[n & 31], w = fma(w0, (double)q, w0);
    return __hiloint2double(__double2hiint(w) - ((n >> 5) << 20), __double2loint(w));
  }
  ATB_DEVICE double exact(float v) const { return !(v > least) ? 0. : top == INFINITY ? 1. : exp_of(((double)v - (double)top) * per_temp); }
};

// What the blocks of a cluster read from each other. A field that others read behind a meeting is written again only behind the next one:
//   top, count, weight      written once
//   first                   set to V before the first meeting, lowered behind it, read behind a second, for a temperature of 0 alone
//   sum                     before the meeting behind the first look, the one behind a sum of what top_k has left, the last one: the meeting of
//                           the lists, or those of an end_of_prefix, lie between a reading and the next
//   above, inside, low, high, least_above, in_bin      before the meeting of a bin, which is followed by another
//   listed                  before the meeting of the lists, and not again: nothing meets between its readers and the first look of the
//                           whole shares
//   few_listed, few, cut    end_of_prefix, whose readings end with a meeting (the first block's `few` is read by itself)
//   best_score, best_at     set before the first meeting, changed by the block's own threads, read behind the last one
// The lists and the parts, in the place of the bins, are read before a meeting that ends their use, too.
struct Shared {
  float top;
  int first;                                     // lowest index of the largest logit
  double sum;                                    // of the weights that this block has
  double above, inside;                          // of those above the bin at hand, and in it
  unsigned long long low, high, least_above;     // keys of the bin at hand, and the least above it
  int in_bin;                                    // tokens in it
  unsigned count[BINS], weight[BINS];            // tokens of a bin, their weights in units of 2^-14 of the bin's largest
  int listed, few_listed;
  unsigned long long few[FEW], cut;
  unsigned long long best_score;                 // fp64 bits
  int best_at;
};

// A row's tokens are shared by the blocks of a cluster, a block's by its threads, which keep them in shared memory where it has room. The loops
// are kept short: a block goes through most of its code once, and has to wait for it.
//
// Without filters every block draws from its share, relative to its own largest logit. With top-k or top-p the end of the prefix is looked
// for first: in a histogram of tokens and weights over the powers of two below the largest weight, where every thread has bins of its own.
// Then every block lists its tokens in the bins down to the one where the prefix ends. If they are few together, the first block puts
// them in order and draws; else all look for the end together, among their lists, and draw from them. Where a block's list would be
// longer than ROOM, they look at their whole shares instead. Looking for the end: the keys' range is divided into SUB parts, and the
// part with the end again, until a few tokens are left, which are put in order and added up. Weights that several threads add up are whole
// numbers (2^-46 of the largest of the range), others are summed in one order, so the result does not depend on which thread comes
// first. A draw is decided in 64 bits: 32-bit arrival times only say which tokens have to be looked at.
// Bound by latency: what a block does one after another. Of 192 rows of 32000 with top-p (62.5 us on the device, 384 blocks in two rounds)
// a block takes 5.5 us for its logits and the largest, 7.3 for the first look, 2.2 and 1.5 to count and to list, 8.7 to find the end,
// 3.7 to draw, 1.8 for the exact look, and 5 in the meetings between; looks after the first only compare a logit, and lists make what
// follows dense (a look that works on every tenth token costs a warp as much as one that works on all). Of 64 rows of 100003 without
// filters (16.5 us) the two looks one behind the other take 6.0 and 6.3, the exact one 2.1, the last meeting 2.4. One row of 32000 with top-k and
// top-p (12.2 us) meets four times, 0.7 to 1.1 us each, and takes 2 us for the first look and as much to count.
template <typename T>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(Args a, int room) {
  // [BINS][THREADS]: weights in the low 22 bits, tokens above; then the list (logit, index), and behind it [4][SUB]: tokens of a part, its
  // weights in three limbs of 16 bits; behind them the share, where there is room
  extern __shared__ __align__(16) unsigned own_bins[];
  int2* const list = reinterpret_cast<int2*>(own_bins);
  unsigned* const parts = own_bins + 2 * ROOM;
  static_assert(ROOM * 8 + 4 * SUB * 4 <= BINS * THREADS * 4, "they lie in the place of the bins");
  __shared__ Shared sh;
  __shared__ double red_d[32];
  __shared__ int red_i[32];
  __shared__ float red_f[33];
  __shared__ double powers[32];
  cg::cluster_group cluster = cg::this_cluster();
  if (threadIdx.x < 32) powers[threadIdx.x] = exp2(threadIdx.x * (-1. / 32.));
  grid_go();
  grid_wait();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31;
  const bool leader = rank == 0;
  const long long row = blockIdx.x / blocks;
  const T* const x = (const T*)a.logits + row * a.stride;
  const float* const wait = a.waiting + row * a.wait_stride;
  // shares begin where the row is aligned to 16 bytes; the first one has what is in front of that
  constexpr int N = Piece<T>::N;
  const int part = ((a.V + blocks - 1) / blocks + 7) / 8 * 8, ahead = (int)(-reinterpret_cast<uintptr_t>(x) & 15) / (int)sizeof(T);
  const int from = rank == 0 ? 0 : min(a.V, rank * part + ahead), to = rank == blocks - 1 ? a.V : min(a.V, (rank + 1) * part + ahead);
  const int body = rank == 0 ? min(ahead, to) : from, pieces = (to - body) / N;
  const double temp = a.t_rows ? a.t_rows[row] : a.t, p = a.p_rows ? a.p_rows[row] : a.p;
  double m = a.m_rows ? a.m_rows[row] : a.m;
  if (m > 1.) m = 1.;
  int k = a.k_rows ? a.k_rows[row] : a.k;
  if (k < 0 || k >= a.V) k = 0;
  const bool failed = *a.status != 0, by_weight = p < 1., unfiltered = k == 0 && !by_weight && !(m > 0.) && temp > 0.;
  // The share's pieces are in shared memory behind the first look, unless there are too many. (From the first-level cache, or L2, every
  // look waited for them anew: 3 us a look where a thread has 8.)
  const bool staged = pieces <= room && !unfiltered;
  uint4* const held = reinterpret_cast<uint4*>(own_bins + BINS * THREADS);
  const uint4* const src = reinterpret_cast<const uint4*>(x + body);
  auto each_odd = [&](auto f) {                  // what lies in no piece: a few at the ends
    const int i = threadIdx.x < 16 ? from + (int)threadIdx.x : body + pieces * N + (int)threadIdx.x - 16;
    if (threadIdx.x < 32 && i < (threadIdx.x < 16 ? body : to)) f(to_f32<T>(x[i]), i);
  };
  auto each_piece = [&](auto f, auto one) {      // f(piece, index of its first), one(logit, index)
    if (staged) {
#pragma unroll 1
      for (int i = threadIdx.x; i < pieces; i += THREADS) f(Piece<T>{held[i]}, body + i * N);
    } else {
#pragma unroll 2
      for (int i = threadIdx.x; i < pieces; i += THREADS) f(Piece<T>{src[i]}, body + i * N);
    }
    each_odd(one);
  };
  auto each = [&](auto f) {                      // f(logit, index)
    each_piece([&](const Piece<T>& v, int i) {
#pragma unroll
                 for (int e = 0; e < N; ++e) f(v[e], i + e);
               }, f);
  };
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
#pragma unroll 4
  for (int i = threadIdx.x; i < pieces; i += THREADS) {      // (a thread reads what it has written itself)
    const Piece<T> v{src[i]};
    if (staged) held[i] = v.u;
    top = fmaxf(top, v.top());
  }
  each_odd([&](float v, int) { top = fmaxf(top, v); });
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
      if (top > -INFINITY) each([&](float v, int i) { if (v == top) first = min(first, i); });
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
  const Scale scale(top, temp, powers);

  // the n <= FEW keys of sh.few in their order, by counting those before each: of this thread's place
  auto put_in_order = [&](int n) {
    const unsigned long long key = (int)threadIdx.x < n ? sh.few[threadIdx.x] : 0;
    int place = n;
    if ((int)threadIdx.x < n) {
      place = 0;
#pragma unroll 8
      for (int i = 0; i < n; ++i) place += sh.few[i] > key;
    }
    __syncthreads();
    if ((int)threadIdx.x < n) sh.few[place] = key;
    __syncthreads();
    return (int)threadIdx.x < n ? sh.few[threadIdx.x] : 0ull;
  };

  // The end of the prefix among the keys that `keys(f)` calls f(key) with in all blocks, those in [low, high], n of them at most: the least
  // key whose predecessors are fewer than `target` tokens (by count), or weigh less. `before` come in front of them.
  auto end_of_prefix = [&](auto keys, unsigned long long low, unsigned long long high, int n, bool count, double target, double before) {
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
        const float v = value_of(key);
        const unsigned long long q = __double2ull_rn(scale.weight<T>(v, scale.power(v)) * per);
        atomicAdd(parts + 1 * SUB + s, (unsigned)q & 0xffffu);
        atomicAdd(parts + 2 * SUB + s, (unsigned)(q >> 16) & 0xffffu);
        atomicAdd(parts + 3 * SUB + s, (unsigned)(q >> 32));
      });
      cluster.sync();
      static_assert(SUB == THREADS, "a thread has one part");
      unsigned mine_n = 0;
      unsigned long long mine_w = 0;
      for (int i = 0; i < blocks; ++i) {
        const unsigned* s = cluster.map_shared_rank(parts, i);
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
      cluster.sync();                            // (the parts have been read by all)
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
    cluster.sync();
    if (leader) {
      n = min(sh.few_listed, FEW);
      for (int r = 1; r < blocks; ++r) {
        const Shared* s = cluster.map_shared_rank(&sh, r);
        const int more = s->few_listed;
        __syncthreads();
        for (int i = threadIdx.x; i < more && n + i < FEW; i += THREADS) sh.few[n + i] = s->few[i];
        n = min(n + more, FEW);
      }
      __syncthreads();
      const unsigned long long key = put_in_order(n);
      double all;
      const double w = (int)threadIdx.x >= n ? 0. : count ? 1. : scale.exact(value_of(key));
      const double till = block_before(w, red_d, all) + before;
      const int left = block_min((int)threadIdx.x < n && till >= target ? (int)threadIdx.x : n);
      if (threadIdx.x == 0) sh.cut = sh.few[max(left, 1) - 1];
    }
    cluster.sync();
    const unsigned long long end = cluster.map_shared_rank(&sh, 0)->cut;
    cluster.sync();
    return end;
  };
  // logits, and keys, of which no token so many powers of two below the largest has a greater one, or a lesser one
  auto floor_at = [&](float y) { return top == INFINITY ? INFINITY : scale.c > 0.f ? fmaxf(scale.top - y / scale.c * 1.00001f, -3.402823466e38f) : -3.402823466e38f; };
  auto lowest_at = [&](float y) { return key_of(floor_at(y), 0xffffffffu); };
  auto highest_at = [&](float y) { return key_of(scale.c > 0.f ? scale.top - y / scale.c * 0.99999f : scale.top, 0); };
  auto score_of = [&](double w, float t) { return t >= 0.f ? quotient_of(w, (double)fabsf(t)) : 0.; };       // (-0 is no time, as 0 is)
  // of the block's threads' tokens the one with the largest score, the lowest of equal ones
  auto best_of_block = [&](double score, int token) {
    if (score >= 0.) atomicMax(&sh.best_score, (unsigned long long)__double_as_longlong(score));
    __syncthreads();
    if (score >= 0. && (unsigned long long)__double_as_longlong(score) == sh.best_score) atomicMin(&sh.best_at, token);
    __syncthreads();
  };

  // The draw: the best arrival in 32 bits, how near the next best of the same thread comes, and the sum of what is left.
  unsigned long long cut = 0;                    // tokens with keys of at least this are left
  double sum = 0.;
  float best = -INFINITY, next = -INFINITY;
  int at = -1;
  bool seen = false;
  auto arrival = [&](float y, float t) { return -y - __log2f(t); };        // (a NaN where t is negative or one: passed over)
  auto arrives = [&](float y, float t, int i) {
    const float s = arrival(y, t);
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
  // what comes first of what the block has seen, looked at exactly, into sh.best_at; `tokens(f)` calls f(logit, index) with all of them.
  // Returns the weights' sum.
  auto come_first = [&](auto tokens) {
    const double all = block_sum(sum, red_d);
    const float block_best = block_max(best, red_f);
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
        tokens([&](float v, int i) {
          const float y = scale.power(v);
          if (y < NOTHING && is_left(v, i) && arrival(y, wait[i]) >= near) look(v, i);
        });
      else
        look(to_f32<T>(x[at]), at);
    }
    best_of_block(score, token);
    if (__syncthreads_or(seen) && sh.best_at == a.V) {
      // none: every waiting time is infinite, or a token without weight arrived at once
      tokens([&](float v, int i) { if (scale.power(v) < NOTHING && is_left(v, i)) look(v, i); });
      best_of_block(score, token);
    }
    return all;
  };

  bool in_lists = false;                         // every block has its tokens that may be left in its list, so many
  int listed = 0;
  if (k > 0 || by_weight) {
    // One look at the row: tokens and weights of the bins, roughly, and with top-p the sum of all weights, which says where the prefix ends
    // as much as the sums in front of a token do; a token without weight does not count.
#pragma unroll
    for (int i = 0; i < BINS; ++i) own_bins[i * THREADS + threadIdx.x] = 0;
    double weights = 0.;
    each([&](float v, int) {
      const float y = scale.power(v);
      if (!(y < NOTHING)) return;
      const int bin = min((int)y, BINS - 1);
      float w;
      if (by_weight) {
        const double exact = scale.weight<T>(v, y);
        weights += exact;
        w = (float)exact;
      } else {
        w = scale.rough(v, y);
      }
      // (w 2^bin lies in (1/2, 1], in the last bin below; 768 = 1.5 * 2^(23 - 14): adding it leaves the nearest unit in the low bits)
      const unsigned q = __float_as_uint(w * __int_as_float((127 + bin) << 23) + 768.f) - __float_as_uint(768.f);
      own_bins[bin * THREADS + threadIdx.x] += (1u << 22) + q;
    });
    const double total_own = block_sum(weights, red_d);
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

    // The block's tokens down to that bin, by their logits alone (and a few beyond, as the bound is rounded): counted, then listed.
    const float until = bin == BINS - 1 ? NOTHING : (float)(bin + 1), floor = floor_at(until);
    int mine = 0, own;
    each([&](float v, int) { mine += v >= floor; });
    int put = block_before(mine, red_i, own);
    if (threadIdx.x == 0) sh.listed = own;
    if (own <= ROOM) {
      each([&](float v, int i) {
        if (v >= floor) list[put++] = make_int2(__float_as_int(v), i);
      });
    }
    cluster.sync();
    const int theirs = lane < blocks ? cluster.map_shared_rank(&sh, lane)->listed : 0;
    const int n = __reduce_add_sync(0xffffffffu, theirs);
    in_lists = __reduce_max_sync(0xffffffffu, theirs) <= ROOM;
    if (n <= FEW) {
      // in their order in the first block, all filters at once
      if (leader) {
        const int r = threadIdx.x >> 5;          // a warp for each block
        int before_r = 0;
        for (int i = 0; i < blocks; ++i) {
          const int u = __shfl_sync(0xffffffffu, theirs, i);
          if (i < r) before_r += u;
        }
        if (r < blocks) {
          const int2* const other = cluster.map_shared_rank(list, r);
          const int more = __shfl_sync(0xffffffffu, theirs, r);
          for (int i = lane; i < more; i += 32) {
            const int2 u = other[i];
            sh.few[before_r + i] = key_of(__int_as_float(u.x), u.y);
          }
        }
        __syncthreads();
        const unsigned long long key = put_in_order(n);
        const int j = threadIdx.x;
        const float v = value_of(key);
        const double w = j < n ? scale.exact(v) : 0.;
        const float t = j < n ? wait[index_of(key)] : 0.f;
        double all;
        const double before = block_before(by_count && j >= k ? 0. : w, red_d, all);
        const double target = by_weight ? p * (by_count ? all : total) : INFINITY;
        const bool behind = j > 0 && (before >= target || w < m);
        const int left = block_min(j >= n || (by_count && j >= k) || behind ? j : THREADS);
        all = block_sum(j < left ? w : 0., red_d);
        const bool drawn = j < left && w > 0.;
        best_of_block(drawn ? score_of(w, t) : -1., drawn ? (int)index_of(key) : a.V);
        if (threadIdx.x == 0) {
          const int i = sh.best_at;
          if (i < a.V) answer(i, log(scale.exact(to_f32<T>(x[i])) / all));
          else answer(0, -INFINITY);
        }
      }
      cluster.sync();                            // the first has read the others' lists
      return;
    }
    if (in_lists) {
      listed = own;
      auto keys = [&](auto f) {
#pragma unroll 2
        for (int i = threadIdx.x; i < own; i += THREADS) f(key_of(__int_as_float(list[i].x), list[i].y));
      };
#pragma unroll 1
      for (int which = by_count ? 0 : 1; which < (by_weight ? 2 : 1); ++which) {
        if (which == 1 && by_count) {            // of what top_k has left
          double s = 0.;
          keys([&](unsigned long long key) { if (key >= cut) s += scale.exact(value_of(key)); });
          s = block_sum(s, red_d);
          if (threadIdx.x == 0) sh.sum = s;
          cluster.sync();
          total = over_blocks(&Shared::sum);
        }
        cut = max(cut, end_of_prefix(keys, max(lowest_at(until), cut), highest_at(0.f), n, which == 0, which == 0 ? (double)k : p * total, 0.));
      }
    }

    // Too many to list: the end in the whole shares.
    for (int which = by_count ? 0 : 1; which < (by_weight ? 2 : 1) && !in_lists; ++which) {
      const bool count = which == 0;
      if (!count && by_count) {                  // of what top_k has left
        double s = 0.;
        each([&](float v, int i) {
          const float y = scale.power(v);
          if (y < NOTHING && key_of(v, i) >= cut) s += scale.weight<T>(v, y);
        });
        const double own = block_sum(s, red_d);
        if (threadIdx.x == 0) sh.sum = own;
        cluster.sync();
        total = over_blocks(&Shared::sum);
      }
      const double target = count ? (double)k : p * total;
      int at_bin = bin;
      if (!count) {
        const unsigned hit = __ballot_sync(0xffffffffu, lane < BINS - 1 && w_to >= target);
        at_bin = min(bin, hit ? __ffs(hit) - 1 : BINS - 1);
      }
      double before = 0.;
      unsigned long long low = 0, high = 0, least_above = ~0ull;
      unsigned inside = 0;
      int way = 0;                               // the bins' rounded weights may be a bin off: up or down from there
      while (true) {
        double w_above = 0., w_inside = 0.;
        unsigned n_above = 0, n_inside = 0;
        unsigned long long lo = ~0ull, hi = 0, over = ~0ull;
        each([&](float v, int i) {
          const float y = scale.power(v);
          if (!(y < NOTHING)) return;
          const int b = min((int)y, BINS - 1);
          const unsigned long long key = key_of(v, i);
          if (b > at_bin || key < cut) return;
          const double w = scale.weight<T>(v, y);
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
        const double above_own = block_sum(count ? (double)n_above : w_above, red_d), inside_own = block_sum(w_inside, red_d);
        if (threadIdx.x == 0) {
          sh.above = above_own;
          sh.inside = inside_own;
          sh.low = sh.least_above = ~0ull;
          sh.high = 0;
          sh.in_bin = 0;
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
          atomicAdd(&sh.in_bin, (int)n_inside);
        }
        cluster.sync();
        const double in = over_blocks(&Shared::inside);
        before = over_blocks(&Shared::above);
        low = least_above = ~0ull;
        high = 0;
        inside = 0;
        for (int i = 0; i < blocks; ++i) {
          const Shared* s = cluster.map_shared_rank(&sh, i);
          inside += s->in_bin;
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
      auto keys = [&](auto f) { each([&](float v, int i) { f(key_of(fmaxf(v, -INFINITY), i)); }); };
      cut = max(cut, end_of_prefix(keys, max(low, cut), high, (int)inside, count, target, before));
    }
  }

  // Every block draws from its share.
  if (unfiltered) {
    // the block's own largest logit says what weights are relative to; for a logarithm rough weights do, a piece's added up in 32 bits
    const bool wide = (reinterpret_cast<uintptr_t>(wait + body) & 15) == 0;
    const float bend = -0.69314718f * scale.c_rest;
    float weights = 0.f;
    auto one = [&](float v, float t, int i) {
      const float y = scale.power(v);
      const float w = fast_exp2(-y);
      weights += fmaf(w, scale.below(v) * bend, w);
      arrives(y, t, i);
    };
#pragma unroll 4
    for (int k = threadIdx.x; k < pieces; k += THREADS) {
      const int i = body + k * N;
      const Piece<T> v{src[k]};
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
      sum += (double)weights;
      weights = 0.f;
    }
    each_odd([&](float v, int i) { one(v, wait[i], i); });
    sum += (double)weights;
  } else if (in_lists) {
    constexpr int EACH = ROOM / THREADS;
    float t[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int j = threadIdx.x + e * THREADS;
      const int2 u = j < listed ? list[j] : make_int2(0, 0);
      t[e] = j < listed && is_left(__int_as_float(u.x), u.y) ? wait[u.y] : -1.f;
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int j = threadIdx.x + e * THREADS;
      if (j >= listed) continue;
      const float v = __int_as_float(list[j].x), y = scale.power(v);
      if (!(y < NOTHING) || !is_left(v, list[j].y)) continue;
      sum += scale.weight<T>(v, y);
      arrives(y, t[e], list[j].y);
    }
  } else {
    const float floor = cut != 0 ? value_of(cut) : m > 0. && scale.top < INFINITY ? scale.top - never : -3.402823466e38f;
    auto drawn = [&](float v, int i) { return v >= floor && scale.power(v) < NOTHING && is_left(v, i); };
    each([&](float v, int i) {
      if (!drawn(v, i)) return;
      const float y = scale.power(v);
      sum += scale.weight<T>(v, y);
      arrives(y, wait[i], i);
    });
  }
  const double sum_own = come_first([&](auto f) {
    if (in_lists)
      for (int i = threadIdx.x; i < listed; i += THREADS) f(__int_as_float(list[i].x), list[i].y);
    else
      each(f);
  });
  if (threadIdx.x == 0) sh.sum = sum_own;
  cluster.sync();
  if (leader && threadIdx.x < 32) {
    // the blocks' tokens relative to the row's largest logit
    const Shared* s = cluster.map_shared_rank(&sh, lane < blocks ? lane : 0);
    const float own = lane < blocks ? s->top : -INFINITY;
    top = warp_max(own);
    const Scale all(top, temp, powers);
    double w = lane < blocks && own > -INFINITY ? s->sum * (unfiltered ? all.exact(own) : 1.) : 0.;
    double weights = 0.;
    for (int r = 0; r < blocks; ++r) weights += __shfl_sync(0xffffffffu, w, r);
    int i = lane < blocks ? s->best_at : a.V;
    w = i < a.V ? all.exact(to_f32<T>(x[i])) : 0.;
    double score = i < a.V && w > 0. ? score_of(w, wait[i]) : -1.;
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
      else answer(i, log(w / weights));
    }
  }
  cluster.sync();
}

template <typename T>
int launch(const Args& a, int rows, cudaStream_t st) {
  constexpr int N = THREADS * (16 / sizeof(T)), BINS_BYTES = BINS * THREADS * 4, MOST = 64 << 10;
  static std::atomic<unsigned long long> allowed{0};       // devices on which the kernel may have its shared memory
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return launched(cudaErrorInvalidDevice);
  const unsigned long long bit = 1ull << (device & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    const int rc = launched(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, BINS_BYTES + MOST));
    if (rc != 0) return rc;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  // Blocks of a row: as many as have a piece for every thread, as long as the GPU holds all of them at once (two an SM), or, with
  // filters, half as many more. Rows of 32000 fp32 with top-p 0.9, us with one, two, four and eight blocks: 1 row 34, 26, 23, 26; 32 rows 85,
  // 29, 30, 37; 64 rows 87, 36, 32, 72; 150 rows 110, 52, 77, 168; 192 rows 127, 66, 92, 208; with top-k 50 besides (bf16) 192 rows 33, 35,
  // 50, 95. Without filters (bf16) 64 rows 11.8, 13.2, 10.0, 17; 150 rows 18, 23, 27, 42; 64 rows of 100003 (two, four, eight) 26, 21,
  // 31. The rule takes one block too early where a list has no room in it: 256 rows with top-p 128, with two 77; 192 rows of 100003 two,
  // 314, with four 174.
  const bool filtered = a.k_rows || a.p_rows || a.m_rows || a.k > 0 || a.p < 1. || a.m > 0.;
  int blocks = 1;
  while (blocks < 8 && (long long)rows * blocks * 2 <= (filtered ? 3 : 2) * 148 && a.V > N * blocks) blocks *= 2;
  // a thread's bins have room for the weights of 255 tokens, a block's parts for those of 65536; they serve top-k and top-p
  while (blocks < 8 && a.V > blocks * 128 * THREADS) blocks *= 2;
  const bool binned = a.k_rows || a.p_rows || a.k > 0 || a.p < 1.;
  if (a.V > (binned ? 8 * 128 * THREADS : 1 << 30) || (long long)rows * blocks > 0x7fffffffLL) return -2;
  const int part = ((a.V + blocks - 1) / blocks + 7) / 8 * 8, bytes = (part + 8) * (int)sizeof(T), room = bytes <= MOST ? bytes : 0;
  return launched(launch_after(sample_kernel<T>, dim3((unsigned)(rows * blocks)), THREADS, BINS_BYTES + room, st, blocks, a, room / 16));
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
