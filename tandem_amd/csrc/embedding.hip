// K5: the embedding lookup with a scale, and its gradient by sorted tokens.
//
//   out[n, :] = s * W[t_n, :]                      (one pass, a copy with a product)
//   dW[v, :]  = s * sum over n with t_n = v of g[n, :],   in the order of n
//
// The gradient is a sum over rows that are strewn over g. The tokens are brought together first (equal tokens side by side, in
// the order of n), then the rows of g are read once each in that order and added in fp32 registers; a row of dW is written
// once, rounded once. No float atomics: the order of every sum is fixed by n, the vocabulary and the width alone.
//
//   1. embedding_sort_kernel: every workgroup reads all tokens and places those of its share of the vocabulary. Of more than 8192 tokens
//      embedding_split_kernel first brings those of a share together, 1024 at a time, and embedding_place_kernel reads its own.
//   2. embedding_sum_kernel: a wave takes a chunk of the sorted entries and a slice of the columns. A token whose entries all lie in
//      the chunk is finished there; one that crosses the chunk's ends leaves fp32 partial sums. The launch's other workgroups
//      write the zeros of the rows that have no token (most rows of a large vocabulary).
//   3. embedding_join_kernel: adds the partial sums of the tokens that cross chunks, in order.
// Small tables and few tokens: embedding_row_kernel alone.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/tandem_hip.h"
#include "common.h"
#include "ops_device.h"

namespace tandem_hip {
namespace ops {

namespace {

// ---------------------------------------------------------------- lookup

constexpr int kLookupThreads = 256;
constexpr int kLookupRows = 4;  // in flight at once

struct LookupArgs {
  const void* weight;
  const void* tokens;
  void* out;
  int64_t n, vocab, dim;
  int vecs;      // accesses per row
  int log_lanes; // lanes per row, as a power of two
  float scale;
};

// A copy with a product, bound by memory: 32768 rows of 2048 bf16 take 39 us, 6.9 TB/s of rows read and written. As many lanes as a row has
// accesses, up to a workgroup; four rows of each are under way at once, since a row's address waits for its token. One row:
// 3.3 us, the launch.
template <typename T, typename I, int kBytes>
__global__ __launch_bounds__(kLookupThreads) void embedding_lookup_kernel(LookupArgs a) {
  constexpr int kN = kBytes / static_cast<int>(sizeof(T));
  using P = Pack<T, kN>;
  const int lanes = 1 << a.log_lanes;
  const int lane = threadIdx.x & (lanes - 1);
  const int rows = kLookupThreads >> a.log_lanes;  // side by side
  const int64_t step = static_cast<int64_t>(gridDim.x) * rows * kLookupRows;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * rows * kLookupRows + (threadIdx.x >> a.log_lanes); base < a.n; base += step) {
    int64_t token[kLookupRows];
#pragma unroll
    for (int r = 0; r < kLookupRows; ++r) {
      const int64_t row = base + r * rows;
      token[r] = row < a.n ? static_cast<int64_t>(static_cast<const I*>(a.tokens)[row]) : 0;
    }
    for (int v = lane; v < a.vecs; v += lanes) {
      P p[kLookupRows];
#pragma unroll
      for (int r = 0; r < kLookupRows; ++r) {
        const bool known = token[r] >= 0 && token[r] < a.vocab;  // a token outside the table reads row 0, and shows
        p[r] = P::load(static_cast<const T*>(a.weight) + (known ? token[r] * a.dim : 0) + static_cast<int64_t>(v) * kN);
      }
#pragma unroll
      for (int r = 0; r < kLookupRows; ++r) {
        const int64_t row = base + r * rows;
        const bool known = token[r] >= 0 && token[r] < a.vocab;
        const float scale = known ? a.scale : __builtin_nanf("");
        float f[kN];
        p[r].get(f);
#pragma unroll
        for (int i = 0; i < kN; ++i) f[i] *= scale;
        p[r].set(f);
        if (row < a.n) p[r].store_nt(static_cast<T*>(a.out) + row * a.dim + static_cast<int64_t>(v) * kN);
      }
    }
  }
}

// ---------------------------------------------------------------- sort

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kMostShare = 512;  // tokens of the vocabulary that one workgroup places: a counter per wave and token in LDS

struct SortArgs {
  const void* tokens;
  uint32_t* keys;    // [entries] the sorted entries' tokens
  uint32_t* order;   // [entries] where they came from
  uint32_t* starts;  // [shares * share + 1] the first entry of every token, see place_of()
  uint32_t vocab, padding;
  uint32_t n, per_wave;  // per_wave: consecutive tokens that a wave reads, whole waves of lanes
  uint32_t share;
  int log_shares;
  void* zero;          // the first bytes of dW, which the launch's other workgroups clear
  int64_t zero_bytes;  // whole vectors from a 16-byte boundary on
};

// Token v belongs to share v mod shares (neighbours, which occur together, are strewn) and is number v / shares in it; the
// sorted order is that of this place.
__host__ __device__ __forceinline__ uint32_t place_of(uint32_t v, uint32_t share, int log_shares) {
  return (v & ((1u << log_shares) - 1)) * share + (v >> log_shares);
}

constexpr uint32_t kNoToken = 0xffffffffu;

// A token that takes no gradient (outside the table, or the padding's) has no key and no entry.
template <typename I>
__device__ __forceinline__ uint32_t key_of(const SortArgs& a, uint32_t n) {
  const I token = static_cast<const I*>(a.tokens)[n];
  const uint32_t low = static_cast<uint32_t>(token);  // negative tokens: either the upper half is not zero or this exceeds any vocabulary
  const bool fits = sizeof(I) == 4 || static_cast<uint32_t>(static_cast<uint64_t>(token) >> 32) == 0;
  return fits && low < a.vocab && low != a.padding ? low : kNoToken;
}

// The zeros that a sort's launch writes beside it.
template <int kThreads>
__device__ __forceinline__ void write_zeros(void* base, int64_t bytes, int64_t block, int64_t blocks) {
  const Vec16 none = {0u, 0u, 0u, 0u};
  Vec16* const to = static_cast<Vec16*>(base);
  for (int64_t v = block * kThreads + threadIdx.x; v < bytes / 16; v += blocks * kThreads) __builtin_nontemporal_store(none, to + v);
}

// Counting sort, a workgroup per share of the vocabulary. Every workgroup reads all tokens (they stay in L2): first it counts those
// of lower shares and, per wave and token, those of its own; after a sum over tokens and waves it knows where each wave's entries
// of each token go, and places them in the order in which they come: a wave walks its stretch of tokens 64 at a
// time, and for every distinct token of its share among the 64 moves that token's counter on once. Any skew is right, and the
// result is the same every time. A lane reads kHeld tokens at once; where they are all its tokens, they stay in registers for
// the second walk. 8192 byte tokens: 10.5 us, bound by the chain of walks, counters and barriers, not by memory. (A radix sort of
// them in one workgroup's LDS took 12.6 us, its merge of four such tiles another 12: one compute unit's instruction rate bound it.)
template <typename I, int kHeld>
__global__ __launch_bounds__(kSortThreads, 8) void embedding_sort_kernel(SortArgs a) {
  if (blockIdx.x >> a.log_shares != 0) {
    const int64_t shares = int64_t(1) << a.log_shares;
    write_zeros<kSortThreads>(a.zero, a.zero_bytes, blockIdx.x - shares, gridDim.x - shares);
    return;
  }
  extern __shared__ uint32_t s_count[];  // [waves][share]
  __shared__ uint32_t s_sum[kSortWaves], s_below[kSortWaves];
  const uint32_t tid = threadIdx.x, lane = tid % kWave;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const uint32_t mine = blockIdx.x, low = (1u << a.log_shares) - 1;
  uint32_t* const count = s_count + wave * a.share;
  const uint32_t first = std::min<uint64_t>(static_cast<uint64_t>(wave) * a.per_wave, a.n);
  const uint32_t end = std::min<uint64_t>(static_cast<uint64_t>(first) + a.per_wave, a.n);
  uint32_t key[kHeld];
  auto read = [&](uint32_t at) {
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const uint32_t n = at + u * kWave + lane;
      key[u] = n < end ? key_of<I>(a, n) : kNoToken;
    }
  };
  // a token's number in this share; kNoToken: it is another's
  auto own = [&](uint32_t k) { return ((k ^ mine) & low) == 0 && k != kNoToken ? k >> a.log_shares : kNoToken; };
  read(first);
  for (uint32_t i = tid; i < kSortWaves * a.share; i += kSortThreads) s_count[i] = 0;
  __syncthreads();

  uint32_t below = 0;
  for (uint32_t at = first; at < end; at += kWave * kHeld) {
    if (at != first) read(at);
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      below += static_cast<uint32_t>(__popcll(__ballot((key[u] & low) < mine)));  // kNoToken is in no lower share
      key[u] = own(key[u]);
      if (key[u] != kNoToken) atomicAdd(&count[key[u]], 1u);
    }
  }
  if (lane == 0) s_below[wave] = below;
  __syncthreads();

  uint32_t of_wave[kSortWaves] = {}, total = 0;
  if (tid < a.share)
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) of_wave[w] = s_count[w * a.share + tid];
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) total += of_wave[w];
  uint32_t upto = total;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint32_t x = __shfl_up(upto, d);
    if (lane >= static_cast<uint32_t>(d)) upto += x;
  }
  if (lane == kWave - 1) s_sum[wave] = upto;
  __syncthreads();
  uint32_t begin = upto - total;
#pragma unroll
  for (uint32_t w = 0; w < kSortWaves; ++w) begin += s_below[w] + (w < wave ? s_sum[w] : 0u);
  if (tid < a.share) {
    a.starts[mine * a.share + tid] = begin;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      s_count[w * a.share + tid] = begin;
      begin += of_wave[w];
    }
    if (mine == low && tid == a.share - 1) a.starts[(low + 1) * a.share] = begin;  // all entries
  }
  __syncthreads();

  for (uint32_t at = first; at < end; at += kWave * kHeld) {
    if (a.per_wave > kWave * kHeld) {
      read(at);
#pragma unroll
      for (int u = 0; u < kHeld; ++u) key[u] = own(key[u]);
    }
    // the counters' answers of four steps are on their way at once: a wave's LDS operations stay in order
    constexpr int kGroup = 4;
#pragma unroll
    for (int v = 0; v < kHeld; v += kGroup) {
      uint32_t found[kGroup], lead[kGroup], rank[kGroup];
#pragma unroll
      for (int u = 0; u < kGroup; ++u) {
        found[u] = lead[u] = rank[u] = 0;
        uint64_t left = __ballot(key[v + u] != kNoToken);
        while (left != 0) {
          const uint32_t leader = static_cast<uint32_t>(__builtin_ctzll(left));
          const uint32_t k = __builtin_amdgcn_readlane(key[v + u], leader);
          const bool same = key[v + u] == k;
          const uint64_t all = __ballot(same);
          if (same) {
            lead[u] = leader;
            rank[u] = static_cast<uint32_t>(__popcll(all & ((1ull << lane) - 1)));
          }
          if (lane == leader) found[u] = atomicAdd(&count[k], static_cast<uint32_t>(__popcll(all)));
          left &= ~all;
        }
      }
#pragma unroll
      for (int u = 0; u < kGroup; ++u) {
        const uint32_t entry = __shfl(found[u], static_cast<int>(lead[u])) + rank[u];
        if (key[v + u] != kNoToken) {
          a.keys[entry] = (key[v + u] << a.log_shares) | mine;
          a.order[entry] = at + (v + u) * kWave + lane;
        }
      }
    }
  }
}

// The same result for many tokens, each read by one workgroup instead of by all (32768 int64 tokens of a vocabulary of 131072: 25 us by 256
// workgroups that all read them, most of it waiting for the same lines; a training step of 2048 columns took 194 us with that, 181 with the split). A tile of tokens is brought in order of their shares, `from`
// where they came from; offsets[tile][share]: where the share's begin in the tile.
constexpr int kSplitThreads = 512, kSplitWaves = kSplitThreads / kWave, kSplitItems = 2, kTile = kSplitThreads * kSplitItems;
constexpr int kPlaceItems = 4;
constexpr int64_t kOneLaunch = 8192;  // tokens that the one launch is quicker with
constexpr int kMostTiles = 1024;  // a workgroup that places holds their numbers in LDS

struct SplitArgs {
  SortArgs sort;
  uint32_t *numbers, *from;  // [n] the token's number in its share; where it stood
  uint32_t* offsets;         // [tiles][shares + 1]
  int tiles, number_bits;
};

// The lanes that hold the same value (of `bits` bits) as this one, among those that take part.
__device__ __forceinline__ uint64_t lanes_like(uint32_t value, int bits, bool takes_part) {
  uint64_t same = __ballot(takes_part);
  for (int b = 0; b < bits; ++b) {
    const bool on = (value >> b) & 1;
    const uint64_t votes = __ballot(on);
    same &= on ? votes : ~votes;
  }
  return same;
}

// Moves the wave's counter of `value` on by the lanes that hold it; every one of them gets its own place: they stay in order.
__device__ __forceinline__ uint32_t claim(uint32_t* count, uint32_t value, int bits, bool takes_part) {
  const uint32_t lane = threadIdx.x % kWave;
  const uint64_t same = lanes_like(value, bits, takes_part);
  const int leader = takes_part ? __builtin_ctzll(same) : 0;
  uint32_t found = 0;
  if (takes_part && lane == static_cast<uint32_t>(leader)) found = atomicAdd(&count[value], static_cast<uint32_t>(__popcll(same)));
  return __shfl(found, leader) + static_cast<uint32_t>(__popcll(same & ((1ull << lane) - 1)));
}

// s_count [waves][width], the number of every wave's entries of every value, becomes where they begin, from `begin` on; returns where
// this lane's value (its number in the workgroup) begins, and in `end` where all end. width: at most the workgroup's lanes.
template <int kWaves>
__device__ __forceinline__ uint32_t begins(uint32_t* s_count, uint32_t width, uint32_t begin, uint32_t& end) {
  __shared__ uint32_t s_sum[kWaves];
  const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  uint32_t of_wave[kWaves] = {}, total = 0;
  if (tid < width)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) of_wave[w] = s_count[w * width + tid];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) total += of_wave[w];
  uint32_t upto = total;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint32_t x = __shfl_up(upto, d);
    if (lane >= static_cast<uint32_t>(d)) upto += x;
  }
  if (lane == kWave - 1) s_sum[wave] = upto;
  __syncthreads();
  end = begin;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    if (w < wave) begin += s_sum[w];
    end += s_sum[w];
  }
  begin += upto - total;
  uint32_t at = begin;
  if (tid < width)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      s_count[w * width + tid] = at;
      at += of_wave[w];
    }
  __syncthreads();
  return begin;
}

template <typename I>
__global__ __launch_bounds__(kSplitThreads) void embedding_split_kernel(SplitArgs a) {
  if (static_cast<int>(blockIdx.x) >= a.tiles) {
    write_zeros<kSplitThreads>(a.sort.zero, a.sort.zero_bytes, static_cast<int64_t>(blockIdx.x) - a.tiles, static_cast<int64_t>(gridDim.x) - a.tiles);
    return;
  }
  extern __shared__ uint32_t s_count[];  // [waves][shares]
  const uint32_t tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const uint32_t shares = 1u << a.sort.log_shares, low = shares - 1, base = blockIdx.x * static_cast<uint32_t>(kTile);
  uint32_t key[kSplitItems], rank[kSplitItems];
#pragma unroll
  for (int u = 0; u < kSplitItems; ++u) {
    const uint32_t n = base + (wave * kSplitItems + u) * kWave + lane;
    key[u] = n < a.sort.n ? key_of<I>(a.sort, n) : kNoToken;
  }
  for (uint32_t i = tid; i < kSplitWaves * shares; i += kSplitThreads) s_count[i] = 0;
  __syncthreads();
  uint32_t* const count = s_count + wave * shares;
#pragma unroll
  for (int u = 0; u < kSplitItems; ++u) rank[u] = claim(count, key[u] & low, a.sort.log_shares, key[u] != kNoToken);
  __syncthreads();
  uint32_t end;
  const uint32_t begin = begins<kSplitWaves>(s_count, shares, 0u, end);
  uint32_t* const offsets = a.offsets + static_cast<int64_t>(blockIdx.x) * (shares + 1);
  if (tid < shares) offsets[tid] = begin;
  if (tid == 0) offsets[shares] = end;
#pragma unroll
  for (int u = 0; u < kSplitItems; ++u)
    if (key[u] != kNoToken) {
      const uint32_t to = base + count[key[u] & low] + rank[u];
      a.numbers[to] = key[u] >> a.sort.log_shares;
      a.from[to] = base + (wave * kSplitItems + u) * kWave + lane;
    }
}

__global__ __launch_bounds__(kSortThreads, 8) void embedding_place_kernel(SplitArgs a) {
  extern __shared__ uint32_t s_count[];  // [waves][share]
  __shared__ uint32_t s_upto[kMostTiles], s_skip[kMostTiles], s_part[2][kSortWaves];
  const uint32_t tid = threadIdx.x, lane = tid % kWave;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const uint32_t mine = blockIdx.x, shares = 1u << a.sort.log_shares, share = a.sort.share;
  // of every tile: how many of its entries are this share's, and where they begin in it (as many entries belong to lower shares)
  uint32_t here = 0, skip = 0;
  if (tid < static_cast<uint32_t>(a.tiles)) {
    const uint32_t* const at = a.offsets + static_cast<int64_t>(tid) * (shares + 1) + mine;
    skip = at[0];
    here = at[1] - skip;
  }
  for (uint32_t i = tid; i < kSortWaves * share; i += kSortThreads) s_count[i] = 0;
  uint32_t upto = here, below = skip;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint32_t x = __shfl_up(upto, d);
    if (lane >= static_cast<uint32_t>(d)) upto += x;
    below += __shfl_xor(below, d);
  }
  if (lane == kWave - 1) {
    s_part[0][wave] = upto;
    s_part[1][wave] = below;
  }
  __syncthreads();
  uint32_t first = 0, all = 0;
  below = 0;
#pragma unroll
  for (uint32_t w = 0; w < kSortWaves; ++w) {
    if (w < wave) first += s_part[0][w];
    all += s_part[0][w];
    below += s_part[1][w];
  }
  s_upto[tid] = first + upto;
  s_skip[tid] = tid * static_cast<uint32_t>(kTile) + skip - (first + upto - here);
  __syncthreads();
  // this share's entry e stands in the first tile that reaches beyond it
  auto place_in_split = [&](uint32_t e) {
    uint32_t lo = 0, hi = static_cast<uint32_t>(a.tiles) - 1;
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (s_upto[mid] <= e) lo = mid + 1;
      else hi = mid;
    }
    return s_skip[lo] + e;
  };
  const uint32_t per_wave = (all + kSortThreads - 1) / kSortThreads * kWave;
  const uint32_t begin = std::min(wave * per_wave, all), end = std::min(begin + per_wave, all);
  uint32_t* const count = s_count + wave * share;
  // four steps held in registers: all there are, unless one share has more than 4096 entries
  uint32_t number[kPlaceItems], from[kPlaceItems];
  auto read = [&](uint32_t at) {
#pragma unroll
    for (int u = 0; u < kPlaceItems; ++u) {
      const uint32_t e = at + u * kWave + lane;
      number[u] = kNoToken;
      if (e < end) {
        const uint32_t i = place_in_split(e);
        number[u] = a.numbers[i];
        from[u] = a.from[i];
      }
    }
  };
  read(begin);
  for (uint32_t at = begin; at < end; at += kWave * kPlaceItems) {
    if (at != begin) read(at);
#pragma unroll
    for (int u = 0; u < kPlaceItems; ++u)
      if (number[u] != kNoToken) atomicAdd(&count[number[u]], 1u);
  }
  __syncthreads();
  uint32_t last;
  const uint32_t start = begins<kSortWaves>(s_count, share, below, last);
  if (tid < share) a.sort.starts[mine * share + tid] = start;
  if (mine == shares - 1 && tid == 0) a.sort.starts[shares * share] = last;
  for (uint32_t at = begin; at < end; at += kWave * kPlaceItems) {
    if (per_wave > kWave * kPlaceItems) read(at);
#pragma unroll
    for (int u = 0; u < kPlaceItems; ++u) {
      const uint32_t to = claim(count, number[u], a.number_bits, number[u] != kNoToken);
      if (number[u] != kNoToken) {
        a.sort.keys[to] = (number[u] << a.sort.log_shares) | mine;
        a.sort.order[to] = from[u];
      }
    }
  }
}

// ---------------------------------------------------------------- sums

constexpr int kSumWaves = 4;  // per workgroup
constexpr int kSumThreads = kSumWaves * kWave;
constexpr int64_t kHiddenBytes = int64_t(48) << 20, kHiddenPerToken = 1536;  // of zeros that the sort's launch writes
constexpr int kZeroBytes = 16384, kZeroRows = 1024;  // of dW, at most, per workgroup that writes zeros

struct SumArgs {
  const void* grad;
  const uint32_t *keys, *order, *starts;
  void* dweight;
  float* partial;  // [chunks][2][pitch]: of the token that the chunk begins inside of, of the token that it ends inside of
  int64_t vocab, dim, pitch;
  uint32_t share;
  int log_shares;
  uint32_t all;       // place of the number of entries in `starts`
  int chunk;          // entries
  int slices;         // of a row
  int vecs;           // accesses per row
  uint32_t sums;      // workgroups that add; the others write zeros
  int64_t zero_from;  // the first row whose zeros are still to be written
  int zero_rows;      // of each workgroup
  float scale;
};

template <typename T, int kBytes>
__device__ void zero_rows(const SumArgs& a) {
  __shared__ uint8_t s_empty[kZeroRows];
  const int64_t first = a.zero_from + static_cast<int64_t>(blockIdx.x - a.sums) * a.zero_rows;
  const int rows = static_cast<int>(std::min<int64_t>(a.zero_rows, a.vocab - first));
  for (int r = threadIdx.x; r < rows; r += kSumThreads) {
    const uint32_t p = place_of(static_cast<uint32_t>(first + r), a.share, a.log_shares);
    s_empty[r] = a.starts[p] == a.starts[p + 1];
  }
  __syncthreads();
  char* const to = static_cast<char*>(a.dweight) + first * a.dim * static_cast<int64_t>(sizeof(T));
  const Vec16 none = {0u, 0u, 0u, 0u};
  const uint32_t row_bytes = static_cast<uint32_t>(a.dim) * static_cast<uint32_t>(sizeof(T));
  const uint32_t bytes = static_cast<uint32_t>(rows) * row_bytes;
  if (kBytes == 16 && a.vecs >= kWave) {  // a wave per row
    for (int r = threadIdx.x / kWave; r < rows; r += kSumWaves) {
      if (!s_empty[r]) continue;
      char* const row = to + static_cast<int64_t>(r) * row_bytes;
      for (uint32_t v = threadIdx.x % kWave; v < static_cast<uint32_t>(a.vecs); v += kWave) __builtin_nontemporal_store(none, reinterpret_cast<Vec16*>(row + v * 16u));
    }
    return;
  }
  // short rows, or rows that start anywhere: whole vectors over the ends of rows where all of their rows are empty
  const uint32_t skip = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to) & 15);  // the first vector begins this far before the rows
  for (uint32_t v = threadIdx.x; v * 16u < skip + bytes; v += kSumThreads) {
    const uint32_t begin = v * 16u < skip ? 0u : v * 16u - skip, end = std::min(v * 16u + 16u - skip, bytes);
    const uint32_t last = (end - 1) / row_bytes;
    uint32_t row = begin / row_bytes;
    bool all = end - begin == 16u;
    for (uint32_t r = row; all && r <= last; ++r) all = s_empty[r];
    if (all) {
      *reinterpret_cast<Vec16*>(to + begin) = none;
      continue;
    }
    for (uint32_t b = begin; b < end; b += sizeof(T)) {
      row = b / row_bytes;
      if (s_empty[row]) *reinterpret_cast<T*>(to + b) = narrow<T>(0.0f);
    }
  }
}

// Bound by memory where the table is large: 32768 rows of 2048 bf16 into 131072, 134 MB read and 439 MB written here, take 103 us, 5.6 TB/s.
// Eight rows of g are under way per wave. Chunks of equal length, not one token's rows each: byte tokens, some of which come
// hundreds of times, keep every wave busy (8192 x 768 fp32 for 256 tokens: 6.5 us for 25 MB, and 4.8 for the join).
template <typename T, int kBytes>
__global__ __launch_bounds__(kSumThreads) void embedding_sum_kernel(SumArgs a) {
  constexpr int kN = kBytes / static_cast<int>(sizeof(T));
  constexpr int kAhead = 8;  // rows in flight
  using P = Pack<T, kN>;
  if (blockIdx.x >= a.sums) {
    zero_rows<T, kBytes>(a);
    return;
  }
  const int lane = threadIdx.x % kWave;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * kSumWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t chunk = task / a.slices;
  const int64_t first = chunk * a.chunk;
  const int64_t all = a.starts[a.all];
  if (first >= all) return;
  const int vec = static_cast<int>(task % a.slices) * kWave + lane;
  const bool active = vec < a.vecs;
  const int64_t col = static_cast<int64_t>(active ? vec : 0) * kN;
  const int count = static_cast<int>(std::min<int64_t>(a.chunk, all - first));

  const uint32_t my_key = lane < count ? a.keys[first + lane] : kNoToken;
  const uint32_t my_row = lane < count ? a.order[first + lane] : 0u;
  const uint32_t before = first > 0 ? a.keys[first - 1] : kNoToken;
  const uint32_t after = first + count < all ? a.keys[first + count] : kNoToken;

  float acc[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) acc[i] = 0.0f;
  uint32_t key = __builtin_amdgcn_readlane(my_key, 0);
  bool open = key == before;  // the token began in an earlier chunk

  auto flush = [&](uint32_t k, bool began_before, bool goes_on) {
    if (!active) return;
    if (began_before || goes_on) {
      Pack<float, kN < 4 ? kN : 4> p;
      float* to = a.partial + (chunk * 2 + (began_before ? 0 : 1)) * a.pitch + col;
#pragma unroll
      for (int i = 0; i < kN; i += 4) {
        p.set(acc + i);
        p.store(to + i);
      }
    } else {
      P p;
      float f[kN];
#pragma unroll
      for (int i = 0; i < kN; ++i) f[i] = acc[i] * a.scale;
      p.set(f);
      p.store(static_cast<T*>(a.dweight) + static_cast<int64_t>(k) * a.dim + col);
    }
  };

  const T* grad = static_cast<const T*>(a.grad) + col;
  for (int e = 0; e < count; e += kAhead) {
    P row[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = std::min(e + u, count - 1);
      row[u] = P::load(grad + static_cast<int64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(my_row, at))) * a.dim);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (e + u < count) {
        const uint32_t k = __builtin_amdgcn_readlane(my_key, e + u);
        if (k != key) {
          flush(key, open, false);
          key = k;
          open = false;
#pragma unroll
          for (int i = 0; i < kN; ++i) acc[i] = 0.0f;
        }
        float f[kN];
        row[u].get(f);
#pragma unroll
        for (int i = 0; i < kN; ++i) acc[i] += f[i];
      }
    }
  }
  flush(key, open, key == after);
}

// A workgroup per chunk and slice of 256 columns: if a token begins in the chunk and goes on behind it, its partial sums, the
// workgroup's waves an eighth of them each.
constexpr int kJoinWaves = 8;
constexpr int kJoinCols = 4 * kWave;

template <typename T>
__global__ __launch_bounds__(kJoinWaves* kWave) void embedding_join_kernel(SumArgs a) {
  __shared__ float s_acc[kJoinWaves][kJoinCols];
  const int64_t chunk = blockIdx.x;
  const int64_t first = chunk * a.chunk, next = first + a.chunk;
  const int64_t all = a.starts[a.all];
  const uint32_t key = a.keys[next - 1];  // next is at most n; an entry behind the last holds anything
  if (next >= all) return;
  const uint32_t place = place_of(key, a.share, a.log_shares);
  const int64_t begin = a.starts[place], end = a.starts[place + 1];
  if (begin < first || end <= next) return;  // it began earlier, or ends here
  const int64_t heads = (end - 1) / a.chunk - chunk;  // chunks behind this one that it reaches into
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int64_t col = static_cast<int64_t>(blockIdx.y) * kJoinCols + lane * 4;
  const int64_t per = (heads + kJoinWaves - 1) / kJoinWaves;
  const int64_t from = chunk + 1 + wave * per, to = std::min(chunk + 1 + heads, from + per);
  using P4 = Pack<float, 4>;
  float acc[4] = {};
  if (col < a.dim) {
    if (wave == 0) P4::load(a.partial + (chunk * 2 + 1) * a.pitch + col).get(acc);
#pragma unroll 8
    for (int64_t c = from; c < to; ++c) {
      float f[4];
      P4::load(a.partial + c * 2 * a.pitch + col).get(f);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += f[i];
    }
  }
  P4 sums;
  sums.set(acc);
  sums.store(&s_acc[wave][lane * 4]);
  __syncthreads();
  const int64_t c = static_cast<int64_t>(blockIdx.y) * kJoinCols + threadIdx.x;
  if (threadIdx.x >= kJoinCols || c >= a.dim) return;
  float sum = s_acc[0][threadIdx.x];
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) sum += s_acc[w][threadIdx.x];
  static_cast<T*>(a.dweight)[static_cast<int64_t>(key) * a.dim + c] = narrow<T>(sum * a.scale);
}

// ---------------------------------------------------------------- small tables

// The whole gradient in one launch, for few rows and tokens: a workgroup per row of dW and slice of its columns reads all tokens, lists the places of
// its own in order, and adds those rows of g, a group of lanes per stretch of the list and the groups' sums in order. A row without a token
// comes out as zeros. Latency bounds it, and with it how often the commonest token comes, since one workgroup's loads add it up: 256 rows
// of 512 floats take 5.3 us for 256 tokens, 7.9 for 4096 and 8.8 with a quarter of them the same (sort, sums and join: 10.8, 12.2 and 12.6).
// 8192 tokens, with twice the steps: 11.5 and 15.0 (16.5 and 17.9), but rows that allow no wide loads 26 (21). With 2048 workgroups
// instead of at most 1024 what every one of them costs shows: 512 rows of 512 floats, 4096 tokens, 14.0 us (12.6).
constexpr int kRowThreads = 512, kRowWaves = kRowThreads / kWave, kRowSteps = 8;
constexpr int kRowTokens = kRowThreads * kRowSteps;

struct RowArgs {
  const void *grad, *tokens;
  void* dweight;
  int64_t dim;
  uint32_t n, per_wave, padding;
  int slices, vecs, log_lanes;
  float scale;
};

template <typename T, typename I, int kBytes>
__global__ __launch_bounds__(kRowThreads) void embedding_row_kernel(RowArgs a) {
  constexpr int kN = kBytes / static_cast<int>(sizeof(T)), kAhead = kBytes >= 8 ? 16 : 32;
  using P = Pack<T, kN>;
  using Sums = Pack<float, kN < 4 ? kN : 4>;
  __shared__ uint16_t s_list[kRowTokens];
  __shared__ uint32_t s_found[kRowWaves];
  __shared__ __attribute__((aligned(16))) float s_acc[kRowThreads * kN];
  const uint32_t tid = threadIdx.x, lane = tid % kWave;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const uint32_t v = blockIdx.x / static_cast<uint32_t>(a.slices), slice = blockIdx.x - v * static_cast<uint32_t>(a.slices);
  const uint32_t first = wave * a.per_wave;
  uint32_t mine = 0, found = 0;  // bit j: this lane's token of step j is the row's
#pragma unroll
  for (uint32_t j = 0; j < kRowSteps; ++j) {
    const uint32_t n = first + j * kWave + lane;
    if (j * kWave < a.per_wave && n < a.n && static_cast<const I*>(a.tokens)[n] == static_cast<I>(v)) mine |= 1u << j;
  }
  if (v == a.padding) mine = 0;
#pragma unroll
  for (uint32_t j = 0; j < kRowSteps; ++j) found += static_cast<uint32_t>(__popcll(__ballot((mine >> j) & 1)));
  if (lane == 0) s_found[wave] = found;
  __syncthreads();
  uint32_t at = 0, all = 0;
#pragma unroll
  for (uint32_t w = 0; w < kRowWaves; ++w) {
    if (w < wave) at += s_found[w];
    all += s_found[w];
  }
  if (found != 0) {
#pragma unroll
    for (uint32_t j = 0; j < kRowSteps; ++j) {
      const uint64_t votes = __ballot((mine >> j) & 1);
      if ((mine >> j) & 1) s_list[at + static_cast<uint32_t>(__popcll(votes & ((1ull << lane) - 1)))] = static_cast<uint16_t>(first + j * kWave + lane);
      at += static_cast<uint32_t>(__popcll(votes));
    }
  }
  __syncthreads();

  const uint32_t lanes = 1u << a.log_lanes, group = tid >> a.log_lanes, groups = kRowThreads >> a.log_lanes;
  const uint32_t vec = slice * lanes + (tid & (lanes - 1));
  const uint32_t per = std::max(1u, (all + groups - 1) / groups), used = (all + per - 1) / per;  // groups that have entries
  const uint32_t end = std::min((group + 1) * per, all);
  float acc[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) acc[i] = 0.0f;
  if (vec < static_cast<uint32_t>(a.vecs)) {
    const T* const grad = static_cast<const T*>(a.grad) + static_cast<int64_t>(vec) * kN;
    uint32_t e = group * per;
    auto add = [&](auto ahead, uint32_t count) {  // the next `count` entries, all under way at once
      P row[ahead.value];
#pragma unroll
      for (uint32_t u = 0; u < ahead.value; ++u) row[u] = P::load(grad + static_cast<int64_t>(s_list[e + std::min(u, count - 1)]) * a.dim);
#pragma unroll
      for (uint32_t u = 0; u < ahead.value; ++u)
        if (u < count) {
          float f[kN];
          row[u].get(f);
#pragma unroll
          for (int i = 0; i < kN; ++i) acc[i] += f[i];
        }
      e += count;
    };
    while (e + kAhead <= end) add(std::integral_constant<int, kAhead>{}, kAhead);
    while (e < end) add(std::integral_constant<int, 4>{}, std::min(4u, end - e));
  }
#pragma unroll
  for (int i = 0; i < kN; i += 4) {
    Sums p;
    p.set(acc + i);
    p.store(s_acc + tid * kN + i);
  }
  __syncthreads();
  const uint32_t cols = lanes * kN;
  const int64_t col = static_cast<int64_t>(slice) * cols + tid;
  if (tid >= cols || col >= a.dim) return;
  float sum = 0.0f;
#pragma unroll 8
  for (uint32_t g = 0; g < used; ++g) sum += s_acc[g * cols + tid];
  static_cast<T*>(a.dweight)[static_cast<int64_t>(v) * a.dim + col] = narrow<T>(sum * a.scale);
}

// ---------------------------------------------------------------- host

constexpr int64_t kMostTokens = int64_t(1) << 28;  // the sums' launch stays below 2^32 lanes

// Whether a gradient is the one launch's: at most 1024 workgroups, a row's 512 bytes each, and 4096 tokens whatever the accesses' width (8192 would
// pay with wide loads only, see the kernel).
bool one_launch(int64_t n, int64_t vocab, int64_t dim, int es) { return n <= kRowTokens && vocab * ((dim * es + 511) / 512) <= 1024; }

constexpr int64_t kMostVocab = int64_t(1) << 24;  // 2^15 workgroups place the tokens

// Entries of a chunk: 64, or fewer as long as there are fewer than 2048 waves of 512 columns.
int chunk_of(int64_t n, int64_t dim) {
  int chunk = 64;
  while (chunk > 16 && n / chunk * ((dim + 511) / 512) < 2048) chunk /= 2;
  return chunk;
}

void check_shape(int64_t n, int64_t vocab, int64_t dim, int dtype) {
  require(operator_dtype(dtype), "embedding: the dtype must be float32, float16 or bfloat16");
  require(n >= 0 && n <= kMostTokens, "embedding: 0 to 2^28 tokens");
  require(vocab >= 1 && vocab <= kMostVocab, "embedding: a vocabulary of 1 to 2^24 rows");
  require(dim >= 1 && dim <= (int64_t(1) << 20), "embedding: rows of 1 to 2^20 elements");
}

void check_index(int index_dtype) {
  require(index_dtype == TDM_I64 || index_dtype == TDM_I32, "embedding: tokens must be int64 or int32");
}

template <class F>
void with_width(int width, F&& f) {
  switch (width) {
    case 16: f(std::integral_constant<int, 16>{}); return;
    case 8: f(std::integral_constant<int, 8>{}); return;
    case 4: f(std::integral_constant<int, 4>{}); return;
    default: f(std::integral_constant<int, 2>{}); return;
  }
}

// 64 shares, or as many more as it takes to keep a share's counters in LDS.
int log_shares_of(int64_t vocab) {
  int log = 6;
  while (((vocab - 1) >> log) >= kMostShare) ++log;
  return log;
}

struct Workspace {  // of the gradient
  int64_t keys, order, starts, partial, numbers, from, offsets, bytes;
  bool split;
  int tiles, log_shares;
  int64_t share, pitch;
};

Workspace workspace_of(int64_t n, int64_t vocab, int64_t dim) {
  Workspace w{};
  auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  if (one_launch(n, vocab, dim, 4)) return w;  // and of any type's
  w.log_shares = log_shares_of(vocab);
  w.share = ((vocab - 1) >> w.log_shares) + 1;
  w.pitch = (dim + 3) / 4 * 4;
  w.keys = take(n * 4);
  w.order = take(n * 4);
  w.starts = take(((w.share << w.log_shares) + 1) * 4);
  // In one launch, split: 8192 tokens 10.5 and 11.3 us (256 rows), 11.4 and 13.1 (131072 rows); 12288 tokens 16.4 and 12.1, 16.0 and 13.9; 65536
  // tokens 67 and 29, 66 and 19. With more shares (more than 2^18 rows) or tiles (more than 2^20 tokens) than LDS holds: one launch, and every
  // share's workgroup reads all tokens.
  w.tiles = static_cast<int>((n + kTile - 1) / kTile);
  w.split = n > kOneLaunch && n <= int64_t(kTile) * kMostTiles && w.log_shares <= 9;
  if (w.split) {
    w.numbers = take(n * 4);
    w.from = take(n * 4);
    w.offsets = take(w.tiles * ((int64_t(1) << w.log_shares) + 1) * 4);
  }
  const int chunk = chunk_of(n, dim);
  const int64_t chunks = (n + chunk - 1) / chunk;
  w.partial = take(chunks > 1 ? chunks * 2 * w.pitch * 4 : 0);
  return w;
}

}  // namespace

}  // namespace ops
}  // namespace tandem_hip

using namespace tandem_hip;
using namespace tandem_hip::ops;

extern "C" {

int tdm_k5_embedding(const void* weight, const void* tokens, int index_dtype, void* out, int64_t n, int64_t vocab, int64_t dim, int dtype,
                     float scale, tdm_stream stream) {
  return guard([&] {
    check_shape(n, vocab, dim, dtype);
    check_index(index_dtype);
    if (n == 0) return;
    require(weight != nullptr && tokens != nullptr && out != nullptr, "embedding: null pointer");
    const int es = dtype == TDM_F32 ? 4 : 2;
    const int width = access_width(reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(dim * es), es);
    LookupArgs a{weight, tokens, out, n, vocab, dim, static_cast<int>(dim * es / width), 0, scale};
    while ((1 << a.log_lanes) < a.vecs && (1 << a.log_lanes) < kLookupThreads) ++a.log_lanes;
    const int rows = (kLookupThreads >> a.log_lanes) * kLookupRows;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((n + rows - 1) / rows, int64_t(1) << 22)));
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      with_width(width, [&](auto w) {
        if constexpr (w.value >= static_cast<int>(sizeof(T))) {
          if (index_dtype == TDM_I64)
            hipLaunchKernelGGL((embedding_lookup_kernel<T, int64_t, w.value>), grid, dim3(kLookupThreads), 0, static_cast<hipStream_t>(stream), a);
          else
            hipLaunchKernelGGL((embedding_lookup_kernel<T, int32_t, w.value>), grid, dim3(kLookupThreads), 0, static_cast<hipStream_t>(stream), a);
        }
      });
    });
    check_launch("embedding_lookup launch");
  });
}

int64_t tdm_k5_embedding_grad_workspace(int64_t n, int64_t vocab, int64_t dim) {
  int64_t bytes = -1;
  guard([&] {
    check_shape(n, vocab, dim, TDM_F32);
    bytes = workspace_of(n, vocab, dim).bytes;
  });
  return bytes;
}

int tdm_k5_embedding_grad(const void* grad, const void* tokens, int index_dtype, void* dweight, void* workspace, int64_t workspace_bytes,
                          int64_t n, int64_t vocab, int64_t dim, int dtype, float scale, int64_t padding, tdm_stream stream) {
  return guard([&] {
    check_shape(n, vocab, dim, dtype);
    check_index(index_dtype);
    require(dweight != nullptr && (n == 0 || (grad != nullptr && tokens != nullptr)), "embedding_grad: null pointer");
    const Workspace ws = workspace_of(n, vocab, dim);
    require(ws.bytes == 0 || (workspace != nullptr && workspace_bytes >= ws.bytes), "embedding_grad: the workspace is smaller than tdm_k5_embedding_grad_workspace says");
    require(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "embedding_grad: the workspace must start on 16 bytes");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char* const base = static_cast<char*>(workspace);
    const int es = dtype == TDM_F32 ? 4 : 2;
    const int width = access_width(reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(dweight) | static_cast<uintptr_t>(dim * es), es);
    const int vecs = static_cast<int>(dim * es / width);
    const uint32_t padding_row = padding >= 0 && padding < vocab ? static_cast<uint32_t>(padding) : kNoToken;
    if (one_launch(n, vocab, dim, es)) {
      RowArgs a{grad, tokens, dweight, dim, static_cast<uint32_t>(n), static_cast<uint32_t>((n + kRowThreads - 1) / kRowThreads * kWave), padding_row, 0, vecs, 3, scale};
      // 8 lanes or more side by side, up to 32, and as many more as 128 columns take
      while ((1 << a.log_lanes) < vecs && (a.log_lanes < 5 || (width / es << a.log_lanes) < 128)) ++a.log_lanes;
      a.slices = (vecs + (1 << a.log_lanes) - 1) >> a.log_lanes;
      const dim3 grid(static_cast<unsigned>(vocab * a.slices));
      with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        with_width(width, [&](auto w) {
          if constexpr (w.value >= static_cast<int>(sizeof(T))) {
            if (index_dtype == TDM_I64) hipLaunchKernelGGL((embedding_row_kernel<T, int64_t, w.value>), grid, dim3(kRowThreads), 0, st, a);
            else hipLaunchKernelGGL((embedding_row_kernel<T, int32_t, w.value>), grid, dim3(kRowThreads), 0, st, a);
          }
        });
      });
      check_launch("embedding_row launch");
      return;
    }

    SortArgs s{};
    s.tokens = tokens;
    s.keys = reinterpret_cast<uint32_t*>(base + ws.keys);
    s.order = reinterpret_cast<uint32_t*>(base + ws.order);
    s.starts = reinterpret_cast<uint32_t*>(base + ws.starts);
    s.vocab = static_cast<uint32_t>(vocab);
    s.padding = padding_row;
    s.n = static_cast<uint32_t>(n);
    s.per_wave = static_cast<uint32_t>((n + kSortThreads - 1) / kSortThreads * kWave);
    s.share = static_cast<uint32_t>(ws.share);
    s.log_shares = ws.log_shares;
    // The sort leaves the memory idle: its launch clears as many rows as are written in about its time, whether they get
    // a token or not. They begin on a vector and end with a row.
    const int64_t row_bytes = dim * es;
    int64_t hidden = std::min(vocab, (kHiddenBytes + n * kHiddenPerToken) / row_bytes);
    if (reinterpret_cast<uintptr_t>(dweight) % 16 != 0) hidden = 0;
    while (hidden * row_bytes % 16 != 0) --hidden;
    s.zero = dweight;
    s.zero_bytes = hidden * row_bytes;
    SumArgs a{};
    a.grad = grad;
    a.keys = s.keys;
    a.order = s.order;
    a.starts = s.starts;
    a.dweight = dweight;
    a.partial = reinterpret_cast<float*>(base + ws.partial);
    a.vocab = vocab;
    a.dim = dim;
    a.pitch = ws.pitch;
    a.share = s.share;
    a.log_shares = s.log_shares;
    a.all = s.share << s.log_shares;
    a.chunk = chunk_of(n, dim);
    a.vecs = vecs;
    a.slices = (a.vecs + kWave - 1) / kWave;
    a.zero_from = hidden;
    a.zero_rows = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kZeroRows, kZeroBytes / row_bytes)));
    a.scale = scale;
    const int64_t chunks = (n + a.chunk - 1) / a.chunk;
    const int64_t sums = (chunks * a.slices + kSumWaves - 1) / kSumWaves;
    const int64_t zeros = (vocab - hidden + a.zero_rows - 1) / a.zero_rows;
    require(sums + zeros < (int64_t(1) << 24), "embedding_grad: too many tokens, rows or columns for one launch");
    a.sums = static_cast<uint32_t>(sums);

    const unsigned shares = 1u << ws.log_shares, zeroing = static_cast<unsigned>(std::min<int64_t>((s.zero_bytes + 65535) / 65536, 1024));
    const unsigned lds = kSortWaves * s.share * 4;
    if (ws.split) {
      SplitArgs p{};
      p.sort = s;
      p.numbers = reinterpret_cast<uint32_t*>(base + ws.numbers);
      p.from = reinterpret_cast<uint32_t*>(base + ws.from);
      p.offsets = reinterpret_cast<uint32_t*>(base + ws.offsets);
      p.tiles = ws.tiles;
      while ((s.share - 1) >> p.number_bits != 0) ++p.number_bits;
      const dim3 grid(static_cast<unsigned>(ws.tiles) + zeroing);
      if (index_dtype == TDM_I64) hipLaunchKernelGGL((embedding_split_kernel<int64_t>), grid, dim3(kSplitThreads), kSplitWaves * shares * 4, st, p);
      else hipLaunchKernelGGL((embedding_split_kernel<int32_t>), grid, dim3(kSplitThreads), kSplitWaves * shares * 4, st, p);
      check_launch("embedding_split launch");
      hipLaunchKernelGGL(embedding_place_kernel, dim3(shares), dim3(kSortThreads), lds, st, p);
      check_launch("embedding_place launch");
    } else {
      const int held = static_cast<int>(s.per_wave / kWave);
      auto sort = [&](auto h) {
        if (index_dtype == TDM_I64) hipLaunchKernelGGL((embedding_sort_kernel<int64_t, h.value>), dim3(shares + zeroing), dim3(kSortThreads), lds, st, s);
        else hipLaunchKernelGGL((embedding_sort_kernel<int32_t, h.value>), dim3(shares + zeroing), dim3(kSortThreads), lds, st, s);
      };
      if (held <= 4) sort(std::integral_constant<int, 4>{});
      else sort(std::integral_constant<int, 8>{});
      check_launch("embedding_sort launch");
    }

    if (sums + zeros == 0) return;
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      with_width(width, [&](auto w) {
        if constexpr (w.value >= static_cast<int>(sizeof(T)))
          hipLaunchKernelGGL((embedding_sum_kernel<T, w.value>), dim3(static_cast<unsigned>(sums + zeros)), dim3(kSumThreads), 0, st, a);
      });
      check_launch("embedding_sum launch");
      if (chunks > 1) {
        hipLaunchKernelGGL((embedding_join_kernel<T>), dim3(static_cast<unsigned>(n / a.chunk), static_cast<unsigned>((dim + kJoinCols - 1) / kJoinCols)),
                           dim3(kJoinWaves * kWave), 0, st, a);
        check_launch("embedding_join launch");
      }
    });
  });
}

}  // extern "C"
