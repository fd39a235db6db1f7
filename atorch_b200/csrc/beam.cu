// One step of a beam search: the best continuations over beams and vocabulary, and the paged cache's move to its new beams.
//
// A continuation of beam w by token v has f = score[w] + (x[w, v] - lse(x[w])), evaluated in fp32 in this order; NaN counts as
// -inf. The `keep` largest f of a sequence's beams are kept, equal ones by the lower w, then the lower v.
#include <atomic>
#include <cooperative_groups.h>
#include "row.cuh"

namespace {
using namespace atb;
namespace cg = cooperative_groups;

// threads of a share of a row, beams, candidates that a share has room for, groups of lanes whose maxima are ranked
constexpr int THREADS = 256, MOST = 32, ROOM = 512, GROUPS = THREADS / 4;

// The same with the beam before the index: the order of a sequence's continuations. 0 is below all of them.
constexpr int INDEX_BITS = 27;
ATB_DEVICE unsigned long long with_beam(unsigned long long key, int beam) {
  if (key == 0) return 0;
  return (key >> 32 << 32) | ((uint32_t)(MOST - 1 - beam) << INDEX_BITS) | ((1u << INDEX_BITS) - 1 - index_of(key));
}
ATB_DEVICE int beam_of(unsigned long long key) { return MOST - 1 - (int)((uint32_t)key >> INDEX_BITS); }
ATB_DEVICE unsigned token_of(unsigned long long key) { return (1u << INDEX_BITS) - 1 - ((uint32_t)key & ((1u << INDEX_BITS) - 1)); }

ATB_DEVICE float total(float score, float x, float lse) {
  const float f = __fadd_rn(score, __fsub_rn(x, lse));
  return f != f ? -INFINITY : f;
}

ATB_DEVICE unsigned long long block_max_key(unsigned long long k, unsigned long long* red) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(0xffffffffu, k, o);
    k = x > k ? x : k;
  }
  __syncthreads();
  if (lane == 0) red[w] = k;
  __syncthreads();
  unsigned long long t = lane < (int)(blockDim.x >> 5) ? red[lane] : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(0xffffffffu, t, o);
    t = x > t ? x : t;
  }
  return t;
}

template <typename T, int P>
using Share = RowShare<T, P, THREADS>;
// Maximum and sum of exponentials relative to it, of two sets
struct Sum {
  float top, sum;
};
ATB_DEVICE Sum add(Sum a, Sum b) {
  const float top = fmaxf(a.top, b.top);
  return Sum{top, a.sum * (a.top == top ? 1.f : expf(a.top - top)) + b.sum * (b.top == top ? 1.f : expf(b.top - top))};
}

struct Out {
  float* scores;
  long long* tokens;
  int* parents;
  unsigned char* ended;
};
// `key`: with its beam. Behind a failed kernel nothing is selected: the first token of the first beam, impossible and ended, so that
// what goes on from there finds indices in range.
ATB_DEVICE void write_out(const Out& out, long long at, unsigned long long key, const unsigned char* ended, int eos, bool failed) {
  if (failed) {
    out.scores[at] = -INFINITY;
    out.tokens[at] = 0;
    out.parents[at] = 0;
    out.ended[at] = 1;
    return;
  }
  out.scores[at] = value_of(key);
  out.tokens[at] = token_of(key);
  out.parents[at] = beam_of(key);
  out.ended[at] = (ended && ended[beam_of(key)]) || (int)token_of(key) == eos;
}
// Place of key number i among n of them (only those that are 0 are equal)
ATB_DEVICE int place_of(const unsigned long long* keys, int n, int i) {
  const unsigned long long k = keys[i];
  int place = 0;
#pragma unroll 4
  for (int j = 0; j < n; ++j) place += keys[j] > k || (keys[j] == k && j < i);
  return place;
}

// The `keep` best continuations of one beam, best first, as keys of f and token; or, where the blocks of all W beams of a sequence
// fit into a cluster (`best` is null, `beams` = W and not 1), those of the sequence at once. The blocks of a cluster have a share of a beam's
// vocabulary each: they add up the row's sum of exponentials through each other's shared memory, each picks the best of its share,
// and the first picks the best of those. The row comes from memory once, and from registers or the first-level cache after that.
// Bound by latency for a few beams (one block a row, with the row's 64 KB read three times from L2, took 17 us).
template <typename T, int P>
__global__ void __launch_bounds__(THREADS, P == 8 ? 3 : 1) beam_row_kernel(const T* logits, const float* scores, const unsigned char* finished,
                                                           unsigned long long* best, Out final, int beams, int V,
                                                           long long row_stride, int wide, int eos, int keep, const int* status) {
  __shared__ Sum warp_sums[THREADS / 32], share_sum;
  __shared__ unsigned long long red_key[THREADS / 32], room[ROOM], tops[GROUPS], mine[MOST];
  __shared__ float least;
  __shared__ int count;
  grid_go();
  grid_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31;
  const int shares = blocks / beams, share_rank = rank % shares, first_rank = rank - share_rank;
  const long long item = blockIdx.x / blocks, row = item * beams + rank / shares;
  const bool failed = *status != 0;      // (the blocks of a cluster stay together)
  const float score = scores[row];
  const bool ended = finished && finished[row];
  // a beam that is not looked at: the end token alone goes on, at no cost, or nothing
  const bool known = ended || score == -INFINITY || score != score;
  const T* x = logits + row * row_stride;
  const int part = ((V + shares - 1) / shares + 7) / 8 * 8, from = min(V, share_rank * part), to = known ? from : min(V, from + part);
  const Share<T, P> share(x, from, to, wide);
  Sum s{-INFINITY, 0.f};
  share.each([&](const Piece<T>& v, int) { s.top = fmaxf(s.top, v.top()); },
             [&](float v, int) { s.top = fmaxf(s.top, v); });
  const float ref = s.top == -INFINITY ? 0.f : s.top, log2e = 1.4426950408889634f;
  // exponentials on the special-function unit, off by 2^-22: a sum of thousands is as near as its fp32 adds. The difference comes
  // before the factor: it is exactly 0 at the maximum, however large that is (rows masked by a type's lowest value).
  share.each([&](const Piece<T>& v, int) {
#pragma unroll
            for (int e = 0; e < Piece<T>::N; ++e) s.sum += fast_exp2((v[e] - ref) * log2e);       // (a NaN makes the sum one)
          }, [&](float v, int) { s.sum += fast_exp2((v - ref) * log2e); });
  const float my_top = s.top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s = add(s, Sum{__shfl_xor_sync(0xffffffffu, s.top, o), __shfl_xor_sync(0xffffffffu, s.sum, o)});
  if (lane == 0) warp_sums[threadIdx.x >> 5] = s;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = warp_sums[0];
    for (int i = 1; i < THREADS / 32; ++i) s = add(s, warp_sums[i]);
    share_sum = s;
  }
  cluster.sync();
  s = *cluster.map_shared_rank(&share_sum, first_rank);
  for (int i = 1; i < shares; ++i) s = add(s, *cluster.map_shared_rank(&share_sum, first_rank + i));
  const float lse = s.top + logf(s.sum);

  // the n-th largest of the maxima of four lanes: no fewer than n continuations of the share reach it
  const int n = min(keep, to - from);
  float group_top = fmaxf(my_top, __shfl_xor_sync(0xffffffffu, my_top, 1));
  group_top = fmaxf(group_top, __shfl_xor_sync(0xffffffffu, group_top, 2));
  if ((lane & 3) == 0) tops[threadIdx.x / 4] = key_of(total(score, group_top, lse), threadIdx.x / 4);
  __syncthreads();
  if (threadIdx.x < GROUPS) {
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < GROUPS; ++i) place += tops[i] > tops[threadIdx.x];
    if (place == max(n, 1) - 1) least = value_of(tops[threadIdx.x]);
  }
  if (threadIdx.x < MOST) {
    const int i = threadIdx.x;
    unsigned long long k = 0;
    if (known && share_rank == 0 && i < min(keep, V)) {      // the others are impossible, and stand in their order
      const bool only = ended && score != -INFINITY && score == score;
      k = !only ? key_of(-INFINITY, i) : i == 0 ? key_of(score, eos) : key_of(-INFINITY, i - 1 < eos ? i - 1 : i);
    }
    mine[i] = k;
  }
  __syncthreads();
  const float reach = known ? -INFINITY : least;
  // f grows with x; an x whose f may round up to `reach` is not further below its x than a few roundings
  float x_reach = (reach - score + lse) - 4.8e-7f * (fabsf(reach) + fabsf(score) + fabsf(lse));
  if (!(x_reach <= 3.4e38f)) x_reach = -INFINITY;          // (a score of +inf)
  auto take = [&](float v, int i) {
    const float f = total(score, v, lse);
    if (f >= reach) {
      const int at = atomicAdd(&count, 1);
      if (at < ROOM) room[at] = key_of(f, i);
    }
  };
  if (reach > -INFINITY)
    share.each([&](const Piece<T>& v, int i) {
              if (v.top() >= x_reach) {
#pragma unroll
                for (int e = 0; e < Piece<T>::N; ++e) take(v[e], i + e);
              }
            }, take);
  __syncthreads();
  const int have = count;
  if (reach > -INFINITY && have <= ROOM) {
    for (int i = threadIdx.x; i < have; i += THREADS) {
      const unsigned long long k = room[i];
      int place = 0;
      for (int j = 0; j < have; ++j) place += room[j] > k;
      if (place < n) mine[place] = k;
    }
  } else {
    // too many reach it, or too few continuations are possible at all: one after another
    unsigned long long last = ~0ull;
    for (int k = 0; k < n; ++k) {
      unsigned long long most = 0;
      auto look = [&](float v, int i) {
        const unsigned long long key = key_of(total(score, v, lse), i);
        if (key < last && key > most) most = key;
      };
      share.each([&](const Piece<T>& v, int i) {
                for (int e = 0; e < Piece<T>::N; ++e) look(v[e], i + e);
              }, look);
      last = block_max_key(most, red_key);
      if (threadIdx.x == 0) mine[k] = last;
    }
  }
  cluster.sync();
  if (rank == 0) {
    const int all = blocks * keep;               // keys of the shares, best first each
    for (int i = threadIdx.x; i < all; i += THREADS)
      room[i] = with_beam(*cluster.map_shared_rank(&mine[i % keep], i / keep), i / keep / shares);
    __syncthreads();
    for (int i = threadIdx.x; i < all; i += THREADS) {
      const int place = place_of(room, all, i);
      if (place >= keep) continue;
      if (best != nullptr) best[row * keep + place] = room[i];
      else if (room[i] != 0) write_out(final, item * keep + place, room[i], finished ? finished + item * beams : nullptr, eos, failed);
    }
  }
  cluster.sync();                                // the first has read the others' keys
}

// The best of a sequence's beams (a block): each of the W keep continuations counts those before it.
__global__ void __launch_bounds__(256) beam_join_kernel(const unsigned long long* best, const unsigned char* finished, Out final,
                                                        int W, int keep, int eos, const int* status) {
  __shared__ unsigned long long all[MOST * MOST];
  grid_go();
  grid_wait();
  const bool failed = *status != 0;
  const long long b = blockIdx.x;
  const int n = W * keep;
  for (int i = threadIdx.x; i < n; i += 256) {
    const unsigned long long k = best[b * n + i];          // (of beam 0, as its cluster knew it)
    all[i] = k == 0 ? 0 : k - ((unsigned long long)(i / keep) << INDEX_BITS);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 256) {
    const int place = place_of(all, n, i);
    if (place < keep && all[i] != 0)
      write_out(final, b * keep + place, all[i], finished ? finished + b * W : nullptr, eos, failed);
  }
}

// The cache follows its beams: row b W + w of the table takes the full pages of row b W + parent[w], and its own last page the
// tokens of that row's last page. A warp has the same places of all rows that move, as many as give its lanes EACH of them, and
// reads them all before it writes any, so the rows may change places. Bound by memory: each token of the last pages that moves
// is read and written once. Measured with 32 layers, 8 heads of 128, 10 tokens in the last page: 24 sequences of 8 beams (57 MB
// written) 28 us, 4.1 TB/s both ways; 48 of 4 26 us; 6 of 32 34 us. Two places a lane took 31, 28 and 47; eight 36, 32 and 37; a
// block in the place of the warp 33, 30 and 36; a thread with its place of all rows 32, 25 and 59.
constexpr int EACH = 4;
__global__ void __launch_bounds__(256) beam_reorder_kernel(uint8_t* codes, uint8_t* scales, int* table, const int* lengths,
                                                           const int* parents, int W, int width, long long table_stride,
                                                           int layers, int pages, long long page_bytes, long long scale_bytes,
                                                           int kv_heads, int page_shift, int token_bytes, int* status) {
  __shared__ int2 sh_rows[MOST], sh_pages[MOST];       // of the rows that move: from and to
  __shared__ int sh_moving;
  grid_go();
  grid_wait();
  const int failed = threadIdx.x == 0 ? *status : 0;
  const long long first = (long long)blockIdx.y * W;
  const int n = lengths[first], full = n >> page_shift, rest = n - (full << page_shift);
  bool good = true;
  if (threadIdx.x < 32) {
    const int w = threadIdx.x, own = w < W ? lengths[first + w] : n, from = w < W ? parents[first + w] : w;
    good = n >= 0 && own == n && full + (rest > 0) <= width && from >= 0 && (from < W || w >= W);
    int2 page = make_int2(0, 0);
    if (good && w < W && rest > 0) {
      page = make_int2(table[(first + from) * table_stride + full], table[(first + w) * table_stride + full]);
      good = min(page.x, page.y) >= 0 && max(page.x, page.y) < pages;
    }
    const unsigned moving = __ballot_sync(0xffffffffu, from != w);
    const int place = __popc(moving & ((1u << w) - 1));
    if (from != w) {
      sh_rows[place] = make_int2(from, w);
      sh_pages[place] = page;
    }
    if (w == 0) sh_moving = __popc(moving);
  }
  if (__syncthreads_or(failed != 0)) return;
  if (__syncthreads_or(!good)) {
    if (threadIdx.x == 0) atomicCAS(status, 0, (int)ATB_ERR_BAD_INDEX);
    return;
  }
  const int moving = sh_moving, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (moving == 0) return;
  const unsigned per_token = token_bytes / 16, per_head = rest * per_token, code_pieces = 2 * kv_heads * per_head;
  const unsigned head_bytes = token_bytes << page_shift;
  const bool is_table = blockIdx.x == gridDim.x - 1;
  // a round is `span` places, of all rows that move
  const unsigned all = is_table ? full : code_pieces + kv_heads * rest;
  if (all == 0) return;
  const unsigned most = EACH * 32 / moving / 4 * 4, rounds = (all + most - 1) / most, span = ((all + rounds - 1) / rounds + 3) / 4 * 4;
  unsigned mine[EACH];            // row and place in the round, of this thread
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const unsigned slot = k * 32 + lane, m = slot / span;
    mine[k] = m << 16 | (slot - m * span);
  }
  if (is_table) {
    for (unsigned round = warp; round < rounds; round += 8) {
      int x[EACH];
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        const unsigned m = mine[k] >> 16, i = round * span + (mine[k] & 0xffff);
        if (m < (unsigned)moving && i < all) x[k] = table[(first + sh_rows[m].x) * table_stride + i];
      }
      __syncwarp();
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        const unsigned m = mine[k] >> 16, i = round * span + (mine[k] & 0xffff);
        if (m < (unsigned)moving && i < all) table[(first + sh_rows[m].y) * table_stride + i] = x[k];
      }
    }
    return;
  }
  // the warps of a sequence take the rounds of all layers in turn
  const unsigned step = (gridDim.x - 1) * 8;
  unsigned layer = (blockIdx.x * 8 + warp) / rounds, round = (blockIdx.x * 8 + warp) % rounds;
  while (layer < (unsigned)layers) {
    uint8_t* const code_page = codes + (long long)layer * pages * page_bytes;
    uint8_t* const scale_page = scales + (long long)layer * pages * scale_bytes;
    uint4 x[EACH];
    unsigned at[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const unsigned m = mine[k] >> 16, i = round * span + (mine[k] & 0xffff);
      if (m >= (unsigned)moving || i >= all) continue;
      if (i < code_pieces) {
        const unsigned h = i / per_head;
        at[k] = h * head_bytes + (i - h * per_head) * 16;
        x[k] = *reinterpret_cast<const uint4*>(code_page + sh_pages[m].x * page_bytes + at[k]);
      } else {
        const unsigned j = i - code_pieces, h = j / rest;
        at[k] = ((h << page_shift) + j - h * rest) * 8;
        *reinterpret_cast<uint2*>(&x[k]) = *reinterpret_cast<const uint2*>(scale_page + sh_pages[m].x * scale_bytes + at[k]);
      }
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const unsigned m = mine[k] >> 16, i = round * span + (mine[k] & 0xffff);
      if (m >= (unsigned)moving || i >= all) continue;
      if (i < code_pieces) *reinterpret_cast<uint4*>(code_page + sh_pages[m].y * page_bytes + at[k]) = x[k];
      else *reinterpret_cast<uint2*>(scale_page + sh_pages[m].y * scale_bytes + at[k]) = *reinterpret_cast<const uint2*>(&x[k]);
    }
    layer += step / rounds;
    round += step % rounds;
    if (round >= rounds) {
      round -= rounds;
      ++layer;
    }
  }
}
// Blocks of a cluster that has all beams of a sequence: more than the 8 that need no leave
constexpr int ONE = 16;
template <typename T, int P>
bool large_clusters() {
  static std::atomic<unsigned long long> allowed{0};       // devices on which the kernel may have them
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  const unsigned long long bit = 1ull << (device & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(beam_row_kernel<T, P>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  return true;
}
}  // namespace

// `best`: workspace, a key for each of B W keep; null: the beams of a sequence are one cluster (W up to 16), which needs none.
extern "C" int atb_beam_select(const void* logits, const void* scores, const void* finished, void* best, void* out_scores,
                               void* tokens, void* parents, void* ended, int B, int W, int V, long long row_stride, int wide,
                               int eos, int keep, int dtype, void* stream, void* status) {
  if (B <= 0 || keep <= 0) return 0;
  if (W < 1 || W > MOST || keep > MOST || V < 1 || V > 1 << INDEX_BITS || (long long)B * W > 0x7fffffffLL / ONE) return -1;
  int shares = 1;      // of 2000 tokens at least, as long as all of them are on the GPU at once
  const bool fused = best == nullptr;
  while (shares < (fused ? ONE : 8) && V >= 4000 * shares && (long long)B * W * shares * 2 <= 4 * 148) shares *= 2;
  if (fused) {
    if (W > ONE) return -1;
    while (shares * W > ONE) shares /= 2;
  }
  const int cluster = fused ? shares * W : shares;
  const Out final{(float*)out_scores, (long long*)tokens, (int*)parents, (unsigned char*)ended};
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t rc = cudaErrorInvalidValue;
  const long long part = (V + shares - 1) / shares + 7, pieces = (part * (dtype == 2 ? 4 : 2) / 16 + THREADS - 1) / THREADS;
#define ROWS_OF(T, P)                                                                                                      \
  {                                                                                                                        \
    if (cluster <= 8 || large_clusters<T, P>())                                                                            \
      rc = launch_after(beam_row_kernel<T, P>, dim3(B * W * shares), THREADS, 0, st, cluster, (const T*)logits,             \
                        (const float*)scores, (const unsigned char*)finished, (unsigned long long*)best, final,             \
                        fused ? W : 1, V, row_stride, wide, eos, keep, (const int*)status);                                 \
  }
#define ROWS(T)                              \
  {                                          \
    if (!wide || pieces > 8 || (pieces > 4 && (long long)B * W * shares > 3 * 148)) ROWS_OF(T, 0) \
    else if (pieces > 4) ROWS_OF(T, 8)       \
    else if (pieces > 2) ROWS_OF(T, 4)       \
    else ROWS_OF(T, 2)                       \
  }
  if (dtype == 0) ROWS(__nv_bfloat16)
  if (dtype == 1) ROWS(__half)
  if (dtype == 2) ROWS(float)
#undef ROWS_OF
#undef ROWS
  if (rc != cudaSuccess || fused) return launched(rc);
  return launched(launch_after(beam_join_kernel, dim3(B), 256, 0, st, 1, (const unsigned long long*)best, (const unsigned char*)finished, final,
                      W, keep, eos, (const int*)status));
}

extern "C" int atb_beam_reorder(void* codes, void* scales, void* table, const void* lengths, const void* parents, int B, int W,
                                int width, long long table_stride, int layers, int pages, int kv_heads, int page_shift,
                                int head_dim, void* stream, void* status) {
  if (B <= 0 || W <= 0) return 0;
  if (W > MOST || B > 65535 || layers > 65534 || head_dim % 32) return -1;
  const int token_bytes = head_dim / 2;
  const long long page_bytes = (2LL * kv_heads * token_bytes) << page_shift, scale_bytes = (8LL * kv_heads) << page_shift;
  const long long most = (2LL * kv_heads * token_bytes / 16 + kv_heads) << page_shift;
  if (page_bytes > 0x7fffffffLL || most > 0x7fffffffLL) return -2;
  // eight blocks an SM where there is work for them, and one of a sequence for the table
  const long long places = EACH * 32 / W / 4 * 4, rounds = (most + places - 1) / places * layers / 8 + 1, want = (148 * 8 + B - 1) / B;
  return launched(launch_after(beam_reorder_kernel, dim3((unsigned)(want < rounds ? want : rounds) + 1, B), 256, 0, (cudaStream_t)stream,
                               1, (uint8_t*)codes, (uint8_t*)scales, (int*)table, (const int*)lengths, (const int*)parents, W,
                               width, table_stride, layers, pages, page_bytes, scale_bytes, kv_heads, page_shift, token_bytes,
                               (int*)status));
}
