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

// Threads of a block; bins of a factor of 2 in weight, the last for all that is less; tokens of which one block finds the end of the
// prefix; bins of a step towards it where there are more
constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 20, ROOM = 2048, SUB = 512;
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

// Weights of a row: exactly, and in 32 bits as a power of two (its exponent, how far below the largest) with what rounding the exponent left.
struct Scale {
  float top, c, c_low;         // log2(e) / T in two parts
  double temp;
  ATB_DEVICE float below(float v) const { return v == top ? 0.f : top - v; }
  ATB_DEVICE double exact(float v) const { return v == top ? 1. : v > -INFINITY ? exp(((double)v - (double)top) / temp) : 0.; }
  ATB_DEVICE float power(float v) const { return below(v) * c; }
  // off by 2^-22 of itself (the special-function unit) and 2^-24 of the distance that rounding the logits' difference leaves
  ATB_DEVICE float weight(float v, float y) const {
    if (!(y < 140.f)) return 0.f;
    const float d = below(v), rest = fmaf(d, c, -y) + d * c_low;
    const float w = fast_exp2(-y);
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
  unsigned sub_count[SUB], sub_low[SUB], sub_high[SUB];
  int listed;
  unsigned long long cut;
  unsigned long long best_score;                 // fp64 bits
  int best_at;
};

// A row's tokens are shared by the blocks of a cluster, a block's by its threads, which keep P pieces in registers.
//
// The end of the prefix is looked for in this order: a histogram of tokens and weights over the powers of two below the largest weight, where
// every thread has bins of its own; if no more than ROOM tokens lie in the bins down to the one where the prefix ends, the first block
// lists and sorts them, finds the end from exact sums in 64 bits, and draws. If there are more, the bin is divided into SUB parts by
// the tokens' place in the order, the one with the end again, until few enough are left, and every block draws from its share.
// Weights that are added up are whole numbers (in units below 2^-30 of a bin's largest) or summed in one order, so the result does not depend on
// which thread comes first. A draw is decided in 64 bits: 32-bit arrival times only say which tokens have to be looked at.
template <typename T, int P>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(Args a) {
  // [BINS][THREADS]: weights in the low 22 bits, tokens above; then the list of keys
  extern __shared__ __align__(16) unsigned own_bins[];
  unsigned long long* const list = reinterpret_cast<unsigned long long*>(own_bins);
  __shared__ Shared sh;
  __shared__ double red_d[32];
  __shared__ int red_i[32];
  __shared__ float red_f[33];
  cg::cluster_group cluster = cg::this_cluster();
  grid_go();
  grid_wait();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31;
  const long long row = blockIdx.x / blocks;
  const T* const x = (const T*)a.logits + row * a.stride;
  const float* const wait = a.waiting + row * a.wait_stride;
  const int part = ((a.V + blocks - 1) / blocks + 7) / 8 * 8, from = min(a.V, rank * part), to = min(a.V, from + part);
  const RowShare<T, P, THREADS> share(x, from, to, (reinterpret_cast<uintptr_t>(x) & 15) == 0);
  auto each = [&](auto f) {                      // f(logit, index); a NaN is taken for -inf
    share.each([&](const Piece<T>& v, int i) {
#pragma unroll
                 for (int e = 0; e < Piece<T>::N; ++e) f(fmaxf(v[e], -INFINITY), i + e);
               }, [&](float v, int i) { f(fmaxf(v, -INFINITY), i); });
  };
  auto again = [&](auto f) {                     // the same from memory, for what happens seldom
#pragma unroll 1
    for (int i0 = from + (int)threadIdx.x * 4; i0 < to; i0 += THREADS * 4)
#pragma unroll 1
      for (int i = i0; i < min(i0 + 4, to); ++i) f(fmaxf(to_f32<T>(x[i]), -INFINITY), i);
  };
  const double temp = a.t_rows ? a.t_rows[row] : a.t, p = a.p_rows ? a.p_rows[row] : a.p, m = a.m_rows ? a.m_rows[row] : a.m;
  int k = a.k_rows ? a.k_rows[row] : a.k;
  if (k < 0 || k >= a.V) k = 0;
  const bool failed = *a.status != 0;

  // the largest logit
  float top = -INFINITY;
  share.each([&](const Piece<T>& v, int) { top = fmaxf(top, v.top()); }, [&](float v, int) { top = fmaxf(top, v); });
  top = block_max(top, red_f);
  if (threadIdx.x == 0) {
    sh.top = top;
    sh.first = a.V;
    sh.listed = 0;
  }
  cluster.sync();
  for (int i = 0; i < blocks; ++i) top = fmaxf(top, cluster.map_shared_rank(&sh, i)->top);
  const bool leader = rank == 0;
  auto answer = [&](int token, double logprob) {
    a.tokens[row] = failed ? 0 : token;
    a.logprobs[row] = failed ? -INFINITY : (float)logprob;
  };
  if (top == -INFINITY || !(temp > 0.)) {
    int first = a.V;
    if (top > -INFINITY) again([&](float v, int i) { if (v == top) first = min(first, i); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
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
  const double c = fmin(1.4426950408889634 / temp, 1e38);
  const Scale scale{top, (float)c, (float)(c - (double)(float)c), temp};

  unsigned long long cut = 0;                    // tokens with keys of at least this are left
  const bool by_count = k > 0, by_weight = p < 1.;
  if (by_count || by_weight) {
    // one look at the row: tokens and weights of the bins, and all weights; a token without weight does not count
    for (int i = 0; i < BINS; ++i) own_bins[i * THREADS + threadIdx.x] = 0;
    float sum = 0.f;
    each([&](float v, int) {
      const float y = scale.power(v);
      if (!(y < NOTHING)) return;
      const int bin = min((int)y, BINS - 1);
      const float w = scale.weight(v, y);
      sum += w;
      const unsigned q = bin < BINS - 1 ? __float2uint_rn(fminf(w * __int_as_float((127 + bin) << 23), 1.f) * 16384.f) : 0u;
      own_bins[bin * THREADS + threadIdx.x] += (1u << 22) + q;
    });
    const double total_own = block_sum(sum, red_d);
    if (threadIdx.x == 0) sh.sum = total_own;
    for (int bin = threadIdx.x >> 5; bin < BINS; bin += WARPS) {
      unsigned n = 0, w = 0;
      for (int i = lane; i < THREADS; i += 32) {
        const unsigned u = own_bins[bin * THREADS + i];
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
    double total = 0.;
    unsigned n_bin = 0;
    double w_bin = 0.;
    for (int i = 0; i < blocks; ++i) {
      const Shared* s = cluster.map_shared_rank(&sh, i);
      total += s->sum;
      if (lane < BINS) {
        n_bin += s->count[lane];
        w_bin += s->weight[lane];
      }
    }
    w_bin *= 1. / 16384.;
    for (int i = 0; i < lane; ++i) w_bin *= 0.5;
    // tokens and weights down to the lane's bin
    unsigned n_to = n_bin;
    double w_to = w_bin;
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
    const bool counts = by_count && (unsigned)k < counted;       // (fewer have weight: top_k leaves them all)
    int bin = BINS - 1;                          // the prefix ends in this bin or before
    if (counts) {
      bin = __ffs(__ballot_sync(0xffffffffu, lane < BINS && n_to >= (unsigned)k)) - 1;
    } else if (by_weight) {
      // (the bins' weights are rounded: a bin more rather than one too few)
      const unsigned hit = __ballot_sync(0xffffffffu, lane < BINS - 1 && w_to >= p * total * 1.0002);
      bin = hit ? __ffs(hit) - 1 : BINS - 1;
    }
    const unsigned listed = __shfl_sync(0xffffffffu, n_to, bin);

    // the end of the prefix among the n listed tokens of the first block, which it sorts: how many are left of them. `before` weighs what
    // comes before the list.
    auto sort_list = [&](int n) {
      int size = 2;
      while (size < n) size *= 2;
      for (int i = n + threadIdx.x; i < size; i += THREADS) list[i] = 0;
      for (int span = 2; span <= size; span *= 2)
        for (int step = span / 2; step > 0; step /= 2) {
          __syncthreads();
          for (int i = threadIdx.x; i < size / 2; i += THREADS) {
            const int at = 2 * i - (i & (step - 1)), other = at + step;
            const unsigned long long u = list[at], v = list[other];
            if ((u < v) == ((at & span) == 0)) {
              list[at] = v;
              list[other] = u;
            }
          }
        }
      __syncthreads();
    };
    // the blocks' tokens that `want` asks for, one list in the first block; returns how many
    auto note = [&](float v, int i) {
      const int at = atomicAdd(&sh.listed, 1);
      if (at < ROOM) list[at] = key_of(v, i);
    };
    auto gather = [&] {
      cluster.sync();
      int n = sh.listed;
      if (leader)
        for (int r = 1; r < blocks; ++r) {
          const int more = cluster.map_shared_rank(&sh, r)->listed;
          const unsigned long long* const other = cluster.map_shared_rank(list, r);
          for (int i = threadIdx.x; i < more && n + i < ROOM; i += THREADS) list[n + i] = other[i];
          n += more;
        }
      return min(n, ROOM);
    };
    constexpr int EACH = ROOM / THREADS;

    if (listed <= ROOM) {
      const float until = (float)(bin + 1);
      each([&](float v, int i) {
        const float y = scale.power(v);
        if (y < NOTHING && (bin == BINS - 1 || y < until)) note(v, i);
      });
      const int n = gather();
      if (leader) {
        sort_list(n);
        double w[EACH], sum = 0., all;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const int j = threadIdx.x * EACH + e;
          w[e] = j < n && !(counts && j >= k) ? scale.exact(value_of(list[j])) : 0.;
          sum += w[e];
        }
        const double before = block_before(sum, red_d, all);
        const double most = p * (counts ? all : total);
        int left = counts ? min(k, n) : n;
#pragma unroll
        for (int e = EACH - 1; e >= 0; --e) {      // the first place that is not left any more
          const int j = threadIdx.x * EACH + e;
          double b = before;
          for (int i = 0; i < e; ++i) b += w[i];
          if (j < n && j > 0 && ((by_weight && b >= most) || w[e] < m)) left = min(left, j);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) left = min(left, __shfl_xor_sync(0xffffffffu, left, o));
        if (lane == 0) red_i[threadIdx.x >> 5] = left;
        if (threadIdx.x == 0) {
          sh.best_score = 0;
          sh.best_at = a.V;
        }
        __syncthreads();
        for (int i = 0; i < WARPS; ++i) left = min(left, red_i[i]);
        sum = 0.;
        double score = -1.;
        int token = a.V;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const int j = threadIdx.x * EACH + e;
          if (j >= left || w[e] == 0.) continue;
          sum += w[e];
          const int i = (int)index_of(list[j]);
          const float t = wait[i];
          const double s = t >= 0.f ? w[e] / (double)t : 0.;
          if (s > score || (s == score && i < token)) {
            score = s;
            token = i;
          }
        }
        sum = block_sum(sum, red_d);
        if (score >= 0.) atomicMax(&sh.best_score, (unsigned long long)__double_as_longlong(score));
        __syncthreads();
        if (score >= 0. && (unsigned long long)__double_as_longlong(score) == sh.best_score) atomicMin(&sh.best_at, token);
        __syncthreads();
        if (threadIdx.x == 0) {
          const int i = sh.best_at;
          answer(i, log(scale.exact(to_f32<T>(x[i])) / sum));
        }
      }
      cluster.sync();                            // the first has read the others' lists
      return;
    }

    // Too many for one block: the end of the prefix by steps. Tokens with keys in [low, high] hold it; `target` tokens or so much weight
    // come down to it, `before` of it lie above. Both selections come one after the other where both are asked for.
    for (int which = counts ? 0 : 1; which < (by_weight ? 2 : 1); ++which) {
      const bool count = which == 0;
      double target = count ? (double)k : p * total, before = 0.;
      int at_bin = bin;
      if (!count && counts) {                    // of what top_k has left
        float s = 0.f;
        again([&](float v, int i) { if (key_of(v, i) >= cut) s += scale.weight(v, scale.power(v)); });
        const double own = block_sum(s, red_d);
        cluster.sync();
        if (threadIdx.x == 0) sh.sum = own;
        cluster.sync();
        total = 0.;
        for (int i = 0; i < blocks; ++i) total += cluster.map_shared_rank(&sh, i)->sum;
        target = p * total;
      }
      if (!count) {
        const unsigned hit = __ballot_sync(0xffffffffu, lane < BINS - 1 && w_to >= target);
        at_bin = min(bin, hit ? __ffs(hit) - 1 : BINS - 1);
      }
      unsigned long long low = 0, high = 0, least_above = ~0ull;
      int way = 0;                               // the bins' rounded weights may be a bin off: up or down from there
      while (true) {
        float above = 0.f, inside = 0.f;
        unsigned n_above = 0;
        unsigned long long lo = ~0ull, hi = 0, over = ~0ull;
        again([&](float v, int i) {
          const unsigned long long key = key_of(v, i);
          const float y = scale.power(v);
          if (!(y < NOTHING) || key < cut) return;
          const int b = min((int)y, BINS - 1);
          if (b > at_bin) return;
          const float w = scale.weight(v, y);
          if (b < at_bin) {
            above += w;
            ++n_above;
            over = min(over, key);
          } else {
            inside += w;
            lo = min(lo, key);
            hi = max(hi, key);
          }
        });
        const double above_own = count ? block_sum((double)n_above, red_d) : block_sum((double)above, red_d), inside_own = block_sum((double)inside, red_d);
        if (threadIdx.x == 0) {
          sh.above = above_own;
          sh.inside = inside_own;
          sh.low = sh.least_above = ~0ull;
          sh.high = 0;
        }
        __syncthreads();
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
          hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
          over = min(over, __shfl_xor_sync(0xffffffffu, over, o));
        }
        if (lane == 0) {
          atomicMin(&sh.low, lo);
          atomicMin(&sh.least_above, over);
          atomicMax(&sh.high, hi);
        }
        cluster.sync();
        double in = 0.;
        before = 0.;
        low = least_above = ~0ull;
        high = 0;
        for (int i = 0; i < blocks; ++i) {
          const Shared* s = cluster.map_shared_rank(&sh, i);
          before += s->above;
          in += s->inside;
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
      // units of the weights: 2^-30 of the bin's largest
      const double unit = ldexp(1., -30 - at_bin);
      int n_inside = 0;
      while (true) {
        const unsigned long long range = high - low;
        const int shift = max(0, 64 - __clzll(range) - 9);      // SUB parts at most
        for (int i = threadIdx.x; i < SUB; i += THREADS) sh.sub_count[i] = sh.sub_low[i] = sh.sub_high[i] = 0;
        __syncthreads();
        again([&](float v, int i) {
          const unsigned long long key = key_of(v, i);
          if (key < low || key > high || key < cut) return;
          const int s = (int)((high - key) >> shift);
          atomicAdd(&sh.sub_count[s], 1u);
          if (!count) {
            const float y = scale.power(v);
            const unsigned q = (unsigned)(fminf(scale.weight(v, y) * __int_as_float((127 + at_bin) << 23), 1.f) * 1073741824.f);
            atomicAdd(&sh.sub_low[s], q & 0xffffu);
            atomicAdd(&sh.sub_high[s], q >> 16);
          }
        });
        cluster.sync();
        static_assert(SUB == THREADS, "a thread has one part");
        unsigned n = 0;
        unsigned long long w = 0;
        for (int i = 0; i < blocks; ++i) {
          const Shared* s = cluster.map_shared_rank(&sh, i);
          n += s->sub_count[threadIdx.x];
          w += s->sub_low[threadIdx.x] + ((unsigned long long)s->sub_high[threadIdx.x] << 16);
        }
        double all;
        const double mine = count ? (double)n : (double)w * unit, till = block_before(mine, red_d, all) + before;
        // the first part at whose end the target is reached, or the last that has tokens
        int hit = n > 0 && till + mine >= target ? (int)threadIdx.x : SUB;
        int last = n > 0 ? (int)threadIdx.x : -1;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          hit = min(hit, __shfl_xor_sync(0xffffffffu, hit, o));
          last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
        }
        __syncthreads();
        if (lane == 0) {
          red_i[threadIdx.x >> 5] = hit;
          red_i[16 + (threadIdx.x >> 5)] = last;
        }
        __syncthreads();
        for (int i = 0; i < WARPS; ++i) {
          hit = min(hit, red_i[i]);
          last = max(last, red_i[16 + i]);
        }
        if (hit == SUB) hit = last;
        __syncthreads();
        if ((int)threadIdx.x == hit) {
          red_d[0] = till;
          red_i[0] = (int)n;
        }
        __syncthreads();
        before = red_d[0];
        n_inside = red_i[0];
        const unsigned long long top_key = high - ((unsigned long long)hit << shift);
        const unsigned long long width = (1ull << shift) - 1;
        low = top_key - low > width ? top_key - width : low;
        high = top_key;
        cluster.sync();                          // the parts have been read by all
        if (n_inside <= ROOM || low == high) break;
      }
      // the few that are left: the last of them that the prefix has
      if (threadIdx.x == 0) sh.listed = 0;
      __syncthreads();
      again([&](float v, int i) {
        const unsigned long long key = key_of(v, i);
        if (key >= low && key <= high && key >= cut) note(v, i);
      });
      const int n = gather();
      if (leader) {
        sort_list(n);
        double w[EACH], sum = 0., all;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const int j = threadIdx.x * EACH + e;
          w[e] = j >= n ? 0. : count ? 1. : scale.exact(value_of(list[j]));
          sum += w[e];
        }
        double till = block_before(sum, red_d, all) + before;
        int left = n;                            // the tokens whose predecessors are less than the target
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const int j = threadIdx.x * EACH + e;
          if (j < n && till >= target) left = min(left, j);
          till += w[e];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) left = min(left, __shfl_xor_sync(0xffffffffu, left, o));
        __syncthreads();
        if (lane == 0) red_i[threadIdx.x >> 5] = left;
        __syncthreads();
        for (int i = 0; i < WARPS; ++i) left = min(left, red_i[i]);
        if (threadIdx.x == 0) sh.cut = list[max(left, 1) - 1];
      }
      cluster.sync();
      cut = max(cut, cluster.map_shared_rank(&sh, 0)->cut);
      if (threadIdx.x == 0) sh.listed = 0;
      cluster.sync();
    }
  }

  // The draw: the best arrival in 32 bits, how near the next best of the same thread comes, and the sum of what is left.
  const double most_below = m > 0. ? -temp * log(m) : INFINITY;       // distance from the largest logit
  const float surely = (float)most_below * (1.f - 1e-6f), never = (float)most_below * (1.f + 1e-6f);
  auto is_left = [&](float v, int i) {
    if (cut != 0 && key_of(v, i) < cut) return false;
    if (!(m > 0.)) return true;
    const float d = scale.below(v);
    return d <= surely || (d <= never && !(scale.exact(v) < m));
  };
  float sum = 0.f, best = -INFINITY, next = -INFINITY;
  int at = -1;
  auto arrival = [&](float y, float t) { return -y - __log2f(t >= 0.f ? t : INFINITY); };
  each([&](float v, int i) {
    const float y = scale.power(v);
    if (!(y < NOTHING) || !is_left(v, i)) return;
    sum += scale.weight(v, y);
    const float s = arrival(y, wait[i]);
    if (s > best || at < 0) {
      next = at < 0 ? -INFINITY : best;
      best = s;
      at = i;
    } else {
      next = fmaxf(next, s);
    }
  });
  const double sum_own = block_sum((double)sum, red_d);
  const float block_best = block_max(at < 0 ? -INFINITY : best, red_f);
  if (threadIdx.x == 0) {
    sh.best_score = 0;
    sh.best_at = a.V;
    sh.sum = sum_own;
  }
  __syncthreads();
  // what may come first when it is looked at exactly
  const float near = block_best - 2e-5f * (2.f + fminf(fabsf(block_best), 1e30f));
  double score = -1.;
  int token = a.V;
  auto look = [&](float v, int i) {
    const double w = scale.exact(v);
    if (w == 0.) return;
    const float t = wait[i];
    const double s = t >= 0.f ? w / (double)t : 0.;
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
      look(fmaxf(to_f32<T>(x[at]), -INFINITY), at);
  }
  if (score >= 0.) atomicMax(&sh.best_score, (unsigned long long)__double_as_longlong(score));
  __syncthreads();
  if (score >= 0. && (unsigned long long)__double_as_longlong(score) == sh.best_score) atomicMin(&sh.best_at, token);
  cluster.sync();
  if (leader && threadIdx.x == 0) {
    double all = 0.;
    unsigned long long s = 0;
    int i = a.V;
    for (int r = 0; r < blocks; ++r) {
      const Shared* o = cluster.map_shared_rank(&sh, r);
      all += o->sum;
      if (o->best_at < a.V && (i == a.V || o->best_score > s || (o->best_score == s && o->best_at < i))) {
        s = o->best_score;
        i = o->best_at;
      }
    }
    answer(i, log(scale.exact(to_f32<T>(x[i])) / all));
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
  while (blocks < 8 && (long long)rows * blocks * 2 <= 148 * 2 && a.V > N * blocks) blocks *= 2;
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
