// Embedding: rows of a table by token, and the table's gradient, which sums
// the rows of equal tokens: they are sorted first, in the tokens' order, and
// summed in pieces and over pieces, so that no sum depends on which workgroup
// comes first. Bound by memory but for
// the sort, which is hidden behind the zeros for words that do not come up.
// 16384 tokens through a table of 65536 x 2048 bf16 and back: 113 us, 27 to 30
// the lookup, 39 the sort and the zeros (268 MB, 6.9 TB/s, half of it into the
// cache behind the second level), 34 the sums, 7 those over pieces.

#include "../../include/cchip_operators.h"
#include "heads.hpp"
#include "operators.hpp"
#include "rows.hpp"

#include <algorithm>
#include <cmath>

namespace cchip {
namespace op {
namespace {

struct EmbeddingArgs {
  const int32_t *ids;
  Rows weight, out, dout, dweight;
  int64_t tokens, vocab, width;
  uint32_t per_row;  // groups of 8 columns
  uint64_t groups;   // of all tokens' rows
  float scale;
  bool accumulate;
  // sorting
  uint2 *from, *to;        // (word, token); null `from`: the ids themselves
  uint32_t *counts, *next;  // [block][kBins] of this pass and the one after; null: there is none
  int blocks, shift;
  uint32_t *totals;  // [group of blocks][kBins]
  int group;         // blocks of a group; 0: each block adds all blocks' counts up
  // sums
  const uint2 *sorted;
  float *partial;  // [piece][first run, last run][width]
  int pieces;
  int lanes;  // threads of a row, a power of two in 4 .. 256; 256 threads have as many pieces at a time as they have room for
};

// A thread has eight columns of a row; four rows a thread took as long for
// 16384 rows of 2048 and 4.4 us in place of 3.1 for 301 of 520.
template <typename W, typename T>
__global__ __launch_bounds__(256) void embed(const EmbeddingArgs a) {
  const uint64_t i = uint64_t(block_index()) * 256 + threadIdx.x;
  if (i >= a.groups) return;
  const uint64_t token = a.groups <= 0xFFFFFFFFu ? uint32_t(i) / a.per_row : i / a.per_row;
  const int64_t col = int64_t(i - token * a.per_row) * 8, id = a.ids[token];
  const int n = a.width - col < 8 ? int(a.width - col) : 8;
  const bool there = id >= 0 && id < a.vocab;
  const Raw8<W> r = load8<W>(row_at<W>(a.weight, there ? id : 0) + col, there ? n : 0);
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = there ? a.scale * float(r.x[j]) : 0.0f;
  store8<T>(row_at<T>(a.out, token) + col, x, n);
}

// ---- sorting tokens by word ------------------------------------------------------

// A stable radix sort, kBits of the word a pass. A block of kBlock tokens is a
// workgroup's; its place in each bin is the sum of what all blocks have of
// the bins before and the blocks before of this one. Up to kAddUp blocks every
// workgroup adds that up for itself from the counts in memory (they are 2 KB a
// block). Beyond that, as such reads grow with the square of the tokens (2^30
// would read 560 TB), two kernels before it do so for groups of blocks.
constexpr int kBits = 9, kBins = 1 << kBits, kSortThreads = 512, kSortWaves = kSortThreads / 64, kEach = 4;
constexpr int kBlock = kSortThreads * kEach;
// Both ways take as long for 192 blocks: 94.5 us, in place of 102, for 128 (262144
// tokens, rows of 64), 134 in place of 129 for 256, 253 and 206 for 512, 4385 and
// 1102 for 4096 (rows of 8). Groups are of 64 blocks, or of more where there
// would be over 1024 of them.
constexpr int kAddUp = 192, kGroup = 64, kGroups = 1024;

__device__ __forceinline__ uint32_t word_of(const EmbeddingArgs &a, int64_t token) {
  const int64_t id = a.ids[token];
  return id >= 0 && id < a.vocab ? uint32_t(id) : uint32_t(a.vocab);  // words that are none come last
}

// Zeros for the whole gradient from some workgroups of a launch: the
// `turn`-th of `turns`.
template <typename W>
__device__ __forceinline__ void clear_gradient(const EmbeddingArgs &a, uint32_t turn, uint32_t turns) {
  if (a.accumulate) return;
  const float zeros[8] = {};
  const uint64_t all = uint64_t(a.vocab) * a.per_row;
  for (uint64_t i = uint64_t(turn) * blockDim.x + threadIdx.x; i < all; i += uint64_t(turns) * blockDim.x) {
    const uint64_t row = all <= 0xFFFFFFFFu ? uint32_t(i) / a.per_row : i / a.per_row;
    const int64_t col = int64_t(i - row * a.per_row) * 8;
    store8<W>(row_at<W>(a.dweight, row) + col, zeros, a.width - col < 8 ? int(a.width - col) : 8);
  }
}

// What the first pass's blocks have in each bin; the workgroups behind them
// clear the gradient and the counts of the passes to come.
template <typename W>
__global__ __launch_bounds__(kSortThreads) void count_words(const EmbeddingArgs a, uint32_t *clear, int64_t clear_words) {
  __shared__ uint32_t bins[kBins];
  const int t = threadIdx.x;
  if (int(blockIdx.x) < a.blocks) {
    for (int i = t; i < kBins; i += kSortThreads) bins[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      const int64_t token = int64_t(blockIdx.x) * kBlock + i * kSortThreads + t;
      if (token < a.tokens) atomicAdd(&bins[word_of(a, token) & (kBins - 1)], 1u);
    }
    __syncthreads();
    for (int i = t; i < kBins; i += kSortThreads) a.counts[int64_t(blockIdx.x) * kBins + i] = bins[i];
    return;
  }
  const uint32_t turn = blockIdx.x - a.blocks, turns = gridDim.x - a.blocks;
  for (int64_t i = int64_t(turn) * kSortThreads + t; i < clear_words; i += int64_t(turns) * kSortThreads) clear[i] = 0;
  clear_gradient<W>(a, turn, turns);
}

// A lane's rank among the wave's items of its digit, those counted before
// included, which it adds these to.
template <int Bits>
__device__ __forceinline__ uint32_t rank_of(bool live, uint32_t digit, uint32_t *counts) {
  const int l = threadIdx.x & 63;
  uint64_t same = __ballot(live);
#pragma unroll
  for (int b = 0; b < Bits; b++) {
    const uint64_t set = __ballot(digit >> b & 1);
    same &= digit >> b & 1 ? set : ~set;
  }
  const uint32_t ahead = uint32_t(__popcll(same & ((uint64_t(1) << l) - 1)));
  uint32_t had = 0;
  if (live) had = counts[digit];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (live && ahead == 0) counts[digit] = had + uint32_t(__popcll(same));
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return had + ahead;
}

// Where the items of the thread's bin begin that row `row` of `rows` rows of
// counts has: behind all rows' of the bins before and the rows' before of this
// one. For all threads of a workgroup; `sums` is in LDS.
__device__ __forceinline__ uint32_t place_of(const uint32_t *counts, int64_t rows, int64_t row, uint32_t (&sums)[kSortWaves]) {
  const int t = threadIdx.x, l = t & 63, w = t >> 6;
  uint32_t before = 0, all = 0;
  for (int64_t r0 = 0; r0 < rows; r0 += 16) {
    uint32_t n[16];
#pragma unroll
    for (int i = 0; i < 16; i++) n[i] = counts[(r0 + i < rows ? r0 + i : r0) * kBins + t];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      if (r0 + i < row) before += n[i];
      if (r0 + i < rows) all += n[i];
    }
  }
  uint32_t upto = all;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t x = __shfl_up(upto, d, 64);
    if (l >= d) upto += x;
  }
  if (l == 63) sums[w] = upto;
  __syncthreads();
  for (int i = 0; i < w; i++) upto += sums[i];
  return upto - all + before;
}

// Many blocks: what a group of them has in each bin, and then each block's
// places in the place of its counts.
__global__ __launch_bounds__(kSortThreads) void sum_groups(const EmbeddingArgs a) {
  const int t = threadIdx.x;
  const int64_t first = int64_t(blockIdx.x) * a.group, end = first + a.group < a.blocks ? first + a.group : a.blocks;
  uint32_t sum = 0;
#pragma unroll 16
  for (int64_t b = first; b < end; b++) sum += a.counts[b * kBins + t];
  a.totals[int64_t(blockIdx.x) * kBins + t] = sum;
}

__global__ __launch_bounds__(kSortThreads) void place_blocks(const EmbeddingArgs a) {
  __shared__ uint32_t sums[kSortWaves];
  const int t = threadIdx.x;
  const int64_t first = int64_t(blockIdx.x) * a.group, end = first + a.group < a.blocks ? first + a.group : a.blocks;
  uint32_t place = place_of(a.totals, gridDim.x, blockIdx.x, sums);
  for (int64_t b0 = first; b0 < end; b0 += 16) {
    uint32_t n[16];
#pragma unroll
    for (int i = 0; i < 16; i++) n[i] = a.counts[(b0 + i < end ? b0 + i : b0) * kBins + t];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      if (b0 + i >= end) break;
      a.counts[(b0 + i) * kBins + t] = place;
      place += n[i];
    }
  }
}

__global__ __launch_bounds__(kSortThreads) void sort_words(const EmbeddingArgs a) {
  __shared__ uint32_t bins[kSortWaves][kBins], base[kBins], sums[kSortWaves];
  static_assert(kBins == kSortThreads, "a thread a bin");
  const int t = threadIdx.x, l = t & 63, w = t >> 6;
  const int64_t block = blockIdx.x;

  base[t] = a.group ? a.counts[block * kBins + t] : place_of(a.counts, a.blocks, block, sums);
#pragma unroll
  for (int i = 0; i < kSortWaves; i++) bins[i][t] = 0;
  __syncthreads();

  // ranks among a wave's equal digits, tokens in order
  uint2 item[kEach];
  uint32_t rank[kEach];
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    const int64_t at = block * kBlock + (w * kEach + i) * 64 + l;
    const bool live = at < a.tokens;
    item[i] = make_uint2(0, 0);
    if (live) item[i] = a.from ? a.from[at] : make_uint2(word_of(a, at), uint32_t(at));
    const uint32_t digit = (item[i].x >> a.shift) & (kBins - 1);
    rank[i] = rank_of<kBits>(live, digit, bins[w]);
  }
  __syncthreads();
  uint32_t waves = base[t];
#pragma unroll
  for (int i = 0; i < kSortWaves; i++) {
    const uint32_t n = bins[i][t];
    bins[i][t] = waves;
    waves += n;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    const int64_t at = block * kBlock + (w * kEach + i) * 64 + l;
    if (at >= a.tokens) continue;
    const uint32_t to = bins[w][(item[i].x >> a.shift) & (kBins - 1)] + rank[i];
    a.to[to] = item[i];
    if (a.next) atomicAdd(&a.next[int64_t(to / kBlock) * kBins + ((item[i].x >> (a.shift + kBits)) & (kBins - 1))], 1u);
  }
}

// All tokens in one workgroup, where they fit into LDS, while the others of
// the launch clear the gradient, which takes longer: 16384 tokens are sorted in
// the 39 us that 268 MB of zeros take, in place of 27 us of their own.
constexpr int kInOne = 16384, kOneThreads = 1024, kOneWaves = kOneThreads / 64, kOneEach = kInOne / kOneThreads;
constexpr int kOneBits = 8, kOneBins = 1 << kOneBits;
constexpr size_t kOneBytes = size_t(kInOne) * sizeof(uint2) + size_t(kOneWaves) * kOneBins * sizeof(uint32_t);

template <typename W>
__global__ __launch_bounds__(kOneThreads) void sort_in_one(const EmbeddingArgs a, int passes) {
  extern __shared__ uint2 held[];  // the items, then the counts of each wave
  __shared__ uint32_t sums[kOneWaves], there;
  if (blockIdx.x) return clear_gradient<W>(a, blockIdx.x - 1, gridDim.x - 1);
  uint32_t(*bins)[kOneBins] = reinterpret_cast<uint32_t(*)[kOneBins]>(held + kInOne);
  const int t = threadIdx.x, l = t & 63, w = t >> 6, count = int(a.tokens);
  const uint32_t none = uint32_t(a.vocab);
  // a wave has as many rounds of 64 tokens side by side
  const int rounds = (count + kOneThreads - 1) / kOneThreads, first = w * rounds * 64 + l;
  uint2 item[kOneEach];
#pragma unroll
  for (int i = 0; i < kOneEach; i++) {
    const int at = first + i * 64;
    item[i] = make_uint2(none, 0);
    if (i < rounds && at < count) item[i] = make_uint2(word_of(a, at), uint32_t(at));
  }
  for (int pass = 0; pass < passes; pass++) {
    for (int i = l; i < kOneBins; i += 64) bins[w][i] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    uint32_t rank[kOneEach];
#pragma unroll
    for (int i = 0; i < kOneEach; i++)
      if (i < rounds) rank[i] = rank_of<kOneBits>(item[i].x != none, item[i].x >> (pass * kOneBits) & (kOneBins - 1), bins[w]);
    __syncthreads();
    uint32_t all = 0, upto = 0;
    if (t < kOneBins) {
      for (int i = 0; i < kOneWaves; i++) all += bins[i][t];
      upto = all;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const uint32_t x = __shfl_up(upto, d, 64);
        if (l >= d) upto += x;
      }
      if (l == 63) sums[w] = upto;
    }
    __syncthreads();
    if (t < kOneBins) {
      for (int i = 0; i < w; i++) upto += sums[i];
      if (t == kOneBins - 1) there = upto;
      uint32_t from = upto - all;
      for (int i = 0; i < kOneWaves; i++) {
        const uint32_t n = bins[i][t];
        bins[i][t] = from;
        from += n;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOneEach; i++)
      if (i < rounds && item[i].x != none) held[bins[w][item[i].x >> (pass * kOneBits) & (kOneBins - 1)] + rank[i]] = item[i];
    __syncthreads();
    // what has no word is dropped here, and comes last as such
#pragma unroll
    for (int i = 0; i < kOneEach; i++)
      if (i < rounds) item[i] = first + i * 64 < int(there) ? held[first + i * 64] : make_uint2(none, 0);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kOneEach; i++)
    if (i < rounds && first + i * 64 < count) a.to[first + i * 64] = item[i];
}

// ---- sums over runs of equal words -------------------------------------------------

// Rows of kPiece sorted tokens, 8 columns a thread, half of them (of f32 a
// quarter) on their way at once. A run that lies in the
// piece is finished here; of one that goes on before or behind it the piece's
// part is left for join_words: before first, behind last, and a piece that is
// all one run's counts as first.
constexpr int kPiece = 32;

template <typename W>
__device__ __forceinline__ void add_row(const EmbeddingArgs &a, uint32_t word, int64_t col, int n, const float (&sum)[8]) {
  W *p = row_at<W>(a.dweight, word) + col;
  float x[8];
  if (a.accumulate) {
    const Raw8<W> r = load8<W>(p, n);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = float(r.x[j]) + a.scale * sum[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = a.scale * sum[j];
  }
  store8<W>(p, x, n);
}

template <typename W, typename T>
__global__ __launch_bounds__(256) void sum_words(const EmbeddingArgs a) {
  extern __shared__ uint2 pieces[];  // [piece][its items, and its neighbours']
  const int t = threadIdx.x & (a.lanes - 1), g = threadIdx.x / a.lanes;
  const int64_t piece = int64_t(block_index()) * (256 / a.lanes) + g;
  uint2 *const items = pieces + g * (kPiece + 2);
  const int64_t at0 = piece * kPiece;
  for (int i = t; i < kPiece + 2; i += a.lanes) {
    const int64_t at = at0 + i - 1;
    items[i] = at >= 0 && at < a.tokens ? a.sorted[at] : make_uint2(0xFFFFFFFFu, 0);
  }
  __syncthreads();
  const int64_t col = (int64_t(blockIdx.z) * a.lanes + t) * 8;
  if (piece >= a.pieces || col >= a.width) return;
  const int n = a.width - col < 8 ? int(a.width - col) : 8;
  const int count = a.tokens - at0 < kPiece ? int(a.tokens - at0) : kPiece;
  float sum[8] = {};
  bool from_before = items[1].x == items[0].x;
  constexpr int kRows = sizeof(T) == 2 ? 16 : 8;
  for (int i0 = 0; i0 < count; i0 += kRows) {
    Raw8<T> r[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      const uint2 item = items[1 + (i0 + i < count ? i0 + i : 0)];
      const bool live = i0 + i < count && item.x < a.vocab;
      if (n == 8) {  // one load and no branch
        r[i] = load8<T>(row_at<T>(a.dout, live ? item.y : items[1].y) + col, 8);
      } else {
        r[i] = load8<T>(row_at<T>(a.dout, item.y) + col, live ? n : 0);
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      if (i0 + i >= count) break;
      const uint32_t word = items[1 + i0 + i].x, after = items[2 + i0 + i].x;
#pragma unroll
      for (int j = 0; j < 8; j++) sum[j] += float(r[i].x[j]);
      const bool last = i0 + i + 1 == count;
      if (word == after && !last) continue;
      if (word < a.vocab) {
        if (from_before || word == after) {
          float *p = a.partial + (piece * 2 + (from_before ? 0 : 1)) * a.width + col;
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (j < n) p[j] = sum[j];
        } else {
          add_row<W>(a, word, col, n, sum);
        }
      }
      from_before = false;
#pragma unroll
      for (int j = 0; j < 8; j++) sum[j] = 0.0f;
    }
  }
}

// Runs that begin in one piece and end in another, by the piece they begin in.
// A word of 45000 of 406000 tokens, rows of 57: 313 us by 8 threads in one
// chain of its 1400 pieces, 26 as the workgroup shares them out.
template <typename W>
__global__ __launch_bounds__(256) void join_words(const EmbeddingArgs a) {
  const int64_t piece = block_index();
  if (piece + 1 >= a.pieces) return;
  const int64_t last = piece * kPiece + kPiece - 1;
  const uint32_t word = a.sorted[last].x;
  if (word >= a.vocab || a.sorted[last + 1].x != word) return;
  // a run that began before this piece and fills it is another workgroup's
  if (piece > 0 && a.sorted[last - kPiece].x == word) return;
  // the piece that it ends in: the last whose first token is the run's, among
  // the next 64 by a lane each, beyond them by halves
  const int64_t at = piece + 2 + (threadIdx.x & 63);
  const uint64_t others = ~__ballot(at < a.pieces && a.sorted[at < a.pieces ? at * kPiece : last].x == word);
  int64_t lo = piece + 1 + (others ? __builtin_ctzll(others) : 64), hi = others ? lo : a.pieces - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) / 2;
    if (a.sorted[mid * kPiece].x == word) lo = mid;
    else hi = mid - 1;
  }
  // its pieces' parts by the groups of threads in turn, then the groups'
  __shared__ float sums[256][8];
  const int t = threadIdx.x & (a.lanes - 1), g = threadIdx.x / a.lanes, groups = 256 / a.lanes;
  const int64_t col = (int64_t(blockIdx.z) * a.lanes + t) * 8;
  const int n = a.width - col < 8 ? int(a.width - col) : 8;
  float sum[8] = {};
  if (n > 0) {
    if (g == 0) {
      const Raw8<float> r = load8<float>(a.partial + (piece * 2 + 1) * a.width + col, n);
#pragma unroll
      for (int j = 0; j < 8; j++) sum[j] = r.x[j];
    }
    for (int64_t i0 = piece + 1 + g; i0 <= lo; i0 += 8 * groups) {
      Raw8<float> r[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int64_t at = i0 + i * groups;
        r[i] = load8<float>(a.partial + (at <= lo ? at : lo) * 2 * a.width + col, at <= lo ? n : 0);
      }
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) sum[j] += r[i].x[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; j++) sums[threadIdx.x][j] = sum[j];
  __syncthreads();
  if (g > 0 || n <= 0) return;
  for (int i = 1; i < groups; i++)
#pragma unroll
    for (int j = 0; j < 8; j++) sum[j] += sums[i * a.lanes + t][j];
  add_row<W>(a, word, col, n, sum);
}

// Few tokens: a workgroup a token, which is done where an earlier one has its
// word and adds up the later ones' rows otherwise, in their order; which they
// are every wave finds for itself. One launch, or two with the zeros, where
// sorting takes three.
constexpr int kFew = 512;

template <typename W>
__global__ __launch_bounds__(256) void clear_words(const EmbeddingArgs a) {
  clear_gradient<W>(a, blockIdx.x, gridDim.x);
}

template <typename W, typename T>
__global__ __launch_bounds__(256) void sum_few(const EmbeddingArgs a) {
  const int l = threadIdx.x & 63, token = blockIdx.x, count = int(a.tokens);
  const uint32_t word = word_of(a, token);
  if (word >= a.vocab) return;
  uint64_t equal[kFew / 64];
#pragma unroll
  for (int i = 0; i < kFew / 64; i++) equal[i] = __ballot(i * 64 + l < count && a.ids[i * 64 + l < count ? i * 64 + l : 0] == int32_t(word));
  const int64_t col = (int64_t(blockIdx.z) * blockDim.x + threadIdx.x) * 8;
  const int n = a.width - col < 8 ? int(a.width - col) : 8;
  bool first = true;
#pragma unroll
  for (int i = 0; i < kFew / 64; i++) {
    const uint64_t before = i * 64 > token ? 0 : token - i * 64 >= 64 ? ~uint64_t(0) : (uint64_t(1) << (token - i * 64)) - 1;
    first = first && !(equal[i] & before);
  }
  if (!first || col >= a.width) return;
  float sum[8] = {};
#pragma unroll
  for (int i = 0; i < kFew / 64; i++) {
    uint64_t left = equal[i];
    while (left) {
      Raw8<T> r[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        r[j] = load8<T>(row_at<T>(a.dout, i * 64 + (left ? __builtin_ctzll(left) : 0)) + col, left ? n : 0);
        left &= left - 1;
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int k = 0; k < 8; k++) sum[k] += float(r[j].x[k]);
    }
  }
  add_row<W>(a, word, col, n, sum);
}

// ---- host ----------------------------------------------------------------------------

struct Layout {
  int passes, one_passes, blocks, group, groups, pieces;
  size_t counts, totals, items, partial;  // bytes
  size_t bytes() const { return counts + totals + 2 * items + partial; }
};

Layout layout_of(const cchip_embedding &op) {
  Layout p = {};
  if (op.tokens <= kFew) return p;
  while (op.vocab >> (p.passes * kBits)) p.passes++;  // words 0 .. vocab
  for (p.one_passes = 1; (op.vocab - 1) >> (p.one_passes * kOneBits);) p.one_passes++;  // words that there are
  p.blocks = int((op.tokens + kBlock - 1) / kBlock);
  if (p.blocks > kAddUp) {
    p.group = std::max(kGroup, (p.blocks + kGroups - 1) / kGroups);
    p.groups = (p.blocks + p.group - 1) / p.group;
  }
  p.totals = size_t(p.groups) * kBins * sizeof(uint32_t);
  p.pieces = int((op.tokens + kPiece - 1) / kPiece);
  p.counts = size_t(p.passes) * p.blocks * kBins * sizeof(uint32_t);
  p.items = (size_t(op.tokens) * sizeof(uint2) + 15) / 16 * 16;
  p.partial = size_t(p.pieces) * 2 * op.width * sizeof(float);
  return p;
}

void check_op(const cchip_embedding *op) {
  const char *who = "embedding";
  if (!op) throw InvalidArgument("embedding: no descriptor");
  check_rows_type(who, op->dtype);
  if (op->weight_dtype != op->dtype && op->weight_dtype != CCHIP_F32)
    throw InvalidArgument("embedding: the table is of the operator's dtype or f32");
  if (op->tokens < 0 || op->tokens > (int64_t(1) << 30)) throw InvalidArgument("embedding: tokens are not in 0 .. 2^30");
  if (op->vocab < 1 || op->vocab > INT32_MAX) throw InvalidArgument("embedding: vocab is not in 1 .. 2^31 - 1");
  if (op->width < 1 || op->width > (int64_t(1) << 20)) throw InvalidArgument("embedding: width is not in 1 .. 2^20");
  if (!std::isfinite(op->scale)) throw InvalidArgument("embedding: scale is not finite");
}

// The table's rows, one of which is a word's, and the tokens', one of which is
// written or read, lie apart; those of two types as far as the first rows show it.
void check_apart(const cchip_embedding &op, const char *out_name, const Rows &out, const char *in_name, const Rows &in, bool table_written) {
  const int64_t rows[] = {op.vocab, op.tokens};
  const int size = op.dtype == CCHIP_F32 ? 4 : 2;
  if (op.weight_dtype != op.dtype) return check_place("embedding", op.dtype, op.tokens, op.width, out_name, out, in_name, in, false);
  if (heads_meet(int(op.width), size, {{1, rows[!table_written], 1}}, {out.p, 0, out.row, 0}, {{1, rows[table_written], 1}}, {in.p, 0, in.row, 0}))
    throw InvalidArgument(strf("embedding: %s is written over %s", out_name, in_name));
}

const int32_t *ids_of(const cchip_embedding_io &io) {
  if (!io.ids) throw InvalidArgument("embedding: no ids");
  if (reinterpret_cast<uintptr_t>(io.ids) % 4) throw InvalidArgument("embedding: ids are not aligned to their elements");
  return io.ids;
}

template <typename F>
void with_types(const cchip_embedding &op, F &&f) {
  with_rows_type(op.dtype, [&](auto t) {
    if (op.weight_dtype == CCHIP_F32) f(float(), t);
    else f(t, t);
  });
}

}  // namespace
}  // namespace op
}  // namespace cchip

using namespace cchip;
using namespace cchip::op;

extern "C" {

int cchip_embedding_forward(const cchip_embedding *op, const cchip_embedding_io *io, void *stream) {
  return guarded([&] {
    const char *who = "embedding";
    check_op(op);
    if (!io) throw InvalidArgument("embedding: no tensors");
    if (op->tokens == 0) return;
    EmbeddingArgs a = {};
    a.ids = ids_of(*io);
    a.weight = rows_of(who, "weight", op->weight_dtype, op->vocab, op->width, io->weight, false, true);
    a.out = rows_of(who, "out", op->dtype, op->tokens, op->width, io->out, true, true);
    check_apart(*op, "out", a.out, "weight", a.weight, false);
    a.tokens = op->tokens;
    a.vocab = op->vocab;
    a.width = op->width;
    a.per_row = uint32_t((op->width + 7) / 8);
    a.groups = uint64_t(op->tokens) * a.per_row;
    if (a.groups > (uint64_t(1) << 39)) throw InvalidArgument("embedding: more than 2^42 elements");
    a.scale = op->scale;
    with_types(*op, [&](auto w, auto t) {
      hipLaunchKernelGGL((embed<decltype(w), decltype(t)>), grid_of(int64_t((a.groups + 255) / 256)), dim3(256), 0, (hipStream_t)stream, a);
    });
    check_launch(who);
  });
}

int cchip_embedding_workspace(const cchip_embedding *op, size_t *bytes) {
  return guarded([&] {
    check_op(op);
    if (bytes) *bytes = layout_of(*op).bytes();
  });
}

int cchip_embedding_backward(const cchip_embedding *op, const cchip_embedding_io *io, void *workspace, size_t workspace_bytes,
                             void *stream) {
  return guarded([&] {
    const char *who = "embedding";
    check_op(op);
    if (!io) throw InvalidArgument("embedding: no tensors");
    EmbeddingArgs a = {};
    a.dweight = rows_of(who, "dweight", op->weight_dtype, op->vocab, op->width, io->dweight, true, true);
    if (op->tokens) {
      a.ids = ids_of(*io);
      a.dout = rows_of(who, "dout", op->dtype, op->tokens, op->width, io->dout, false, true);
      check_apart(*op, "dweight", a.dweight, "dout", a.dout, true);
    }
    const Layout p = layout_of(*op);
    if (workspace_bytes < p.bytes() || (p.bytes() && (!workspace || !aligned16(workspace))))
      throw InvalidArgument(strf("embedding: the workspace needs %zu bytes aligned to 16, has %zu", p.bytes(), workspace ? workspace_bytes : 0));
    a.tokens = op->tokens;
    a.vocab = op->vocab;
    a.width = op->width;
    a.per_row = uint32_t((op->width + 7) / 8);
    a.scale = op->scale;
    a.accumulate = io->accumulate != 0;
    a.blocks = p.blocks;
    a.pieces = p.pieces;
    char *at = static_cast<char *>(workspace);
    uint32_t *counts = reinterpret_cast<uint32_t *>(at);
    a.totals = reinterpret_cast<uint32_t *>(at + p.counts);
    a.group = p.group;
    at += p.counts + p.totals;
    uint2 *items[2] = {reinterpret_cast<uint2 *>(at), reinterpret_cast<uint2 *>(at + p.items)};
    a.partial = reinterpret_cast<float *>(at + 2 * p.items);
    const size_t pass_words = size_t(p.blocks) * kBins;
    hipStream_t s = (hipStream_t)stream;
    const int64_t fill = a.accumulate ? 0 : op->vocab * int64_t(a.per_row);
    const auto turns = [&](int64_t work, int threads) { return unsigned(std::min<int64_t>(2048, (work + threads - 1) / threads)); };
    const int threads = int(std::min<int64_t>(256, (int64_t(a.per_row) + 63) / 64 * 64));
    const unsigned columns = unsigned((a.per_row + threads - 1) / threads);
    if (op->tokens <= kFew) {
      with_types(*op, [&](auto w, auto t) {
        typedef decltype(w) W;
        typedef decltype(t) T;
        if (fill) hipLaunchKernelGGL((clear_words<W>), dim3(turns(fill, 256)), dim3(256), 0, s, a);
        check_launch(who);
        if (op->tokens) hipLaunchKernelGGL((sum_few<W, T>), dim3(unsigned(op->tokens), 1, columns), dim3(threads), 0, s, a);
      });
      check_launch(who);
      return;
    }
    if (op->tokens <= kInOne) {
      a.to = items[0];
      with_types(*op, [&](auto w, auto) {
        typedef decltype(w) W;
        allow_lds<&sort_in_one<W>>(int(kOneBytes), who);
        hipLaunchKernelGGL((sort_in_one<W>), dim3(1 + turns(fill, kOneThreads)), dim3(kOneThreads), kOneBytes, s, a, p.one_passes);
      });
      check_launch(who);
    } else {
      const int64_t clear = int64_t(p.passes - 1) * pass_words;
      a.counts = counts;
      with_types(*op, [&](auto w, auto) {
        hipLaunchKernelGGL((count_words<decltype(w)>), dim3(unsigned(p.blocks) + std::max(1u, turns(std::max(clear, fill), kSortThreads))), dim3(kSortThreads), 0, s, a,
                           counts + pass_words, clear);
      });
      check_launch(who);
      for (int i = 0; i < p.passes; i++) {
        a.from = i ? items[(i - 1) & 1] : nullptr;
        a.to = items[i & 1];
        a.counts = counts + i * pass_words;
        a.next = i + 1 < p.passes ? a.counts + pass_words : nullptr;
        a.shift = i * kBits;
        if (p.groups) {
          hipLaunchKernelGGL(sum_groups, dim3(unsigned(p.groups)), dim3(kSortThreads), 0, s, a);
          check_launch(who);
          hipLaunchKernelGGL(place_blocks, dim3(unsigned(p.groups)), dim3(kSortThreads), 0, s, a);
          check_launch(who);
        }
        hipLaunchKernelGGL(sort_words, dim3(unsigned(p.blocks)), dim3(kSortThreads), 0, s, a);
        check_launch(who);
      }
    }
    a.sorted = a.to;
    a.lanes = 4;
    while (a.lanes < 256 && uint32_t(a.lanes) < a.per_row) a.lanes *= 2;
    const int at_once = 256 / a.lanes;
    dim3 grid = grid_of((p.pieces + at_once - 1) / at_once), join_grid = grid_of(p.pieces);
    grid.z = join_grid.z = unsigned((a.per_row + a.lanes - 1) / a.lanes);
    with_types(*op, [&](auto w, auto t) {
      typedef decltype(w) W;
      typedef decltype(t) T;
      hipLaunchKernelGGL((sum_words<W, T>), grid, dim3(256), size_t(at_once) * (kPiece + 2) * sizeof(uint2), s, a);
      check_launch(who);
      if (p.pieces > 1) hipLaunchKernelGGL((join_words<W>), join_grid, dim3(256), 0, s, a);
    });
    check_launch(who);
  });
}

}  // extern "C"
