// K5: the embedding lookup with a scale, and its gradient by sorted tokens.
//
//   out[n, :] = s * W[t_n, :]                      (one pass, a copy with a product)
//   dW[v, :]  = s * sum over n with t_n = v of g[n, :],   in the order of n
//
// The gradient is a sum over rows that are strewn over g. The tokens are sorted first (stable, so that every row of dW
// adds its terms in the order of n, run after run), then the rows of g are read once each, in sorted order, and added in
// fp32 registers; a row of dW is written once, rounded once. No float atomics: the sums' order is fixed by n, the
// vocabulary and the width alone.
//
//   1. embedding_sort_kernel: a workgroup sorts a tile of tokens in LDS; the launch's other workgroups write the zeros of dW
//      meanwhile (most rows of a large vocabulary get no token).
//   2. embedding_merge_kernel (more than one tile): eight sorted runs become one, every entry finding its own place.
//   3. embedding_sum_kernel: a wave takes a chunk of sorted entries and a slice of the columns. A token whose entries all lie in
//      the chunk is finished there; one that crosses the chunk's ends leaves fp32 partial sums.
//   4. embedding_join_kernel: adds the partial sums of the tokens that cross chunks, in order.

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

struct LookupArgs {
  const void* weight;
  const void* tokens;
  void* out;
  int64_t n, vocab, dim;
  int vecs;      // accesses per row
  int log_lanes; // lanes per row, as a power of two
  float scale;
};

template <typename T, typename I, int kBytes>
__global__ __launch_bounds__(kLookupThreads) void embedding_lookup_kernel(LookupArgs a) {
  constexpr int kN = kBytes / static_cast<int>(sizeof(T));
  using P = Pack<T, kN>;
  const int lanes = 1 << a.log_lanes;
  const int lane = threadIdx.x & (lanes - 1);
  const int rows = kLookupThreads >> a.log_lanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * rows;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * rows + (threadIdx.x >> a.log_lanes); row < a.n; row += step) {
    const int64_t token = static_cast<int64_t>(static_cast<const I*>(a.tokens)[row]);
    const bool known = token >= 0 && token < a.vocab;
    const T* from = static_cast<const T*>(a.weight) + (known ? token * a.dim : 0);
    T* to = static_cast<T*>(a.out) + row * a.dim;
    for (int v = lane; v < a.vecs; v += lanes) {
      P p;
      if (known) {
        p = P::load(from + static_cast<int64_t>(v) * kN);
#pragma unroll
        for (int i = 0; i < kN; ++i) p.v[i] = narrow<T>(widen(p.v[i]) * a.scale);
      } else {  // a token outside the table reads nothing, and shows
#pragma unroll
        for (int i = 0; i < kN; ++i) p.v[i] = narrow<T>(__builtin_nanf(""));
      }
      p.store(to + static_cast<int64_t>(v) * kN);
    }
  }
}

// ---------------------------------------------------------------- sort

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortItems = 8;                             // per lane
constexpr int kTile = kSortThreads * kSortItems;          // tokens that one workgroup sorts
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kMergeWays = 8;

struct SortArgs {
  const void* tokens;
  uint32_t* keys;     // [n] sorted within every tile
  uint32_t* order;    // [n] where the key came from
  void* zero;         // dW
  int64_t zero_bytes;
  int64_t n, vocab, padding;
  int tiles;
  int passes, digit_bits;
};

// The token as a sort key: a token that takes no gradient (outside the table, or the padding's) gets the key `vocab`, behind
// all others.
template <typename I>
__device__ __forceinline__ uint32_t key_of(const SortArgs& a, int64_t n) {
  const int64_t token = static_cast<int64_t>(static_cast<const I*>(a.tokens)[n]);
  return static_cast<uint32_t>(token >= 0 && token < a.vocab && token != a.padding ? token : a.vocab);
}

__device__ void write_zeros(char* base, int64_t bytes, int64_t block, int64_t blocks) {
  typedef uint32_t vec16 __attribute__((ext_vector_type(4)));
  const int64_t head = std::min<int64_t>(bytes, (16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15);
  const int64_t body = (bytes - head) / 16;
  const vec16 none = {0u, 0u, 0u, 0u};
  vec16* at = reinterpret_cast<vec16*>(base + head);
  for (int64_t v = block * kSortThreads + threadIdx.x; v < body; v += blocks * kSortThreads) at[v] = none;
  if (block == 0) {  // the bytes before the first and behind the last whole vector: whole elements of two bytes
    const int64_t tail = (bytes - head - body * 16) / 2;
    if (threadIdx.x < head / 2) reinterpret_cast<uint16_t*>(base)[threadIdx.x] = 0;
    if (threadIdx.x < tail) reinterpret_cast<uint16_t*>(base + head + body * 16)[threadIdx.x] = 0;
  }
}

// A tile by least significant digits, in LDS. A wave owns 512 consecutive entries, 64 at a time: the lanes with the same
// digit find each other by ballots, the lowest of them moves the wave's count of that digit on, and an entry's rank is the
// count it found there plus the lanes of its kind below it: stable, and the same every time.
template <typename I>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(SortArgs a) {
  if (static_cast<int>(blockIdx.x) >= a.tiles) {
    write_zeros(static_cast<char*>(a.zero), a.zero_bytes, static_cast<int64_t>(blockIdx.x) - a.tiles, static_cast<int64_t>(gridDim.x) - a.tiles);
    return;
  }
  __shared__ uint32_t s_key[kTile];
  __shared__ uint16_t s_from[kTile];
  __shared__ uint32_t s_count[kSortWaves][kDigits];
  __shared__ uint32_t s_wave[kSortWaves];
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile;
  const int here = static_cast<int>(std::min<int64_t>(kTile, a.n - base));

  uint32_t key[kSortItems];
  uint16_t from[kSortItems];
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int e = wave * (kSortItems * kWave) + r * kWave + lane;
    from[r] = static_cast<uint16_t>(e);
    key[r] = e < here ? key_of<I>(a, base + e) : 0xffffffffu;  // behind everything in every pass: it stays last
  }
  const int digits = 1 << a.digit_bits;
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.digit_bits;
    for (int i = tid; i < kSortWaves * kDigits; i += kSortThreads) (&s_count[0][0])[i] = 0;
    __syncthreads();
    uint32_t rank[kSortItems];
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
      const uint32_t d = (key[r] >> shift) & (digits - 1);
      uint64_t same = ~0ull;
      for (int b = 0; b < a.digit_bits; ++b) {
        const bool on = (d >> b) & 1;
        const uint64_t votes = __ballot(on);
        same &= on ? votes : ~votes;
      }
      const int leader = __ffsll(static_cast<unsigned long long>(same)) - 1;
      uint32_t found = 0;
      if (lane == leader) found = atomicAdd(&s_count[wave][d], static_cast<uint32_t>(__popcll(same)));
      found = __shfl(found, leader);
      rank[r] = found + static_cast<uint32_t>(__popcll(same & ((1ull << lane) - 1)));
    }
    __syncthreads();
    // where each wave's entries of each digit begin: an exclusive sum over digits, and over waves within a digit
    uint32_t total = 0, mine = 0;
    if (tid < digits)
      for (int w = 0; w < kSortWaves; ++w) total += s_count[w][tid];
    mine = total;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const uint32_t below = __shfl_up(mine, d);
      if (lane >= d) mine += below;
    }
    if (lane == kWave - 1) s_wave[wave] = mine;
    __syncthreads();
    uint32_t begin = mine - total;
    for (int w = 0; w < wave; ++w) begin += s_wave[w];
    if (tid < digits)
      for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t c = s_count[w][tid];
        s_count[w][tid] = begin;
        begin += c;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
      const uint32_t d = (key[r] >> shift) & (digits - 1);
      const uint32_t to = s_count[wave][d] + rank[r];
      s_key[to] = key[r];
      s_from[to] = from[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
      const int e = wave * (kSortItems * kWave) + r * kWave + lane;
      key[r] = s_key[e];
      from[r] = s_from[e];
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kSortItems; ++r) {
    const int e = wave * (kSortItems * kWave) + r * kWave + lane;
    if (e < here) {
      a.keys[base + e] = key[r];
      a.order[base + e] = static_cast<uint32_t>(base + from[r]);
    }
  }
}

// Eight sorted runs of `run` entries become one: an entry's place is its own index plus, for every other run of its group,
// the number of that run's entries that go before it (equal keys of an earlier run do, of a later one do not: stable).
struct MergeArgs {
  const uint32_t *keys, *order;
  uint32_t *to_keys, *to_order;
  int64_t n, run;
};

__global__ __launch_bounds__(256) void embedding_merge_kernel(MergeArgs a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= a.n) return;
  const uint32_t key = a.keys[i];
  const int64_t group = i / (a.run * kMergeWays) * (a.run * kMergeWays);
  const int64_t own = (i - group) / a.run;
  int64_t place = i - (group + own * a.run);
  for (int r = 0; r < kMergeWays; ++r) {
    if (r == own) continue;
    const int64_t begin = group + r * a.run;
    if (begin >= a.n) break;
    int64_t lo = begin, hi = std::min<int64_t>(begin + a.run, a.n);
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      const uint32_t k = a.keys[mid];
      if (r < own ? k <= key : k < key) lo = mid + 1;
      else hi = mid;
    }
    place += lo - begin;
  }
  a.to_keys[group + place] = key;
  a.to_order[group + place] = a.order[i];
}

// ---------------------------------------------------------------- sums

constexpr int kSumWaves = 4;  // per workgroup

struct SumArgs {
  const void* grad;
  const uint32_t *keys, *order;
  void* dweight;
  float* partial;  // [chunks][2][dim]: of the token that the chunk begins inside of, of the token that it ends inside of
  int64_t n, vocab, dim;
  int chunk;   // entries
  int slices;  // of a row
  int vecs;    // accesses per row
  float scale;
};

template <typename T, int kBytes>
__global__ __launch_bounds__(kSumWaves * kWave) void embedding_sum_kernel(SumArgs a) {
  constexpr int kN = kBytes / static_cast<int>(sizeof(T));
  constexpr int kAhead = 8;  // rows in flight
  using P = Pack<T, kN>;
  const int lane = threadIdx.x % kWave;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * kSumWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t chunk = task / a.slices;
  const int64_t first = chunk * a.chunk;
  if (first >= a.n) return;
  const int vec = static_cast<int>(task % a.slices) * kWave + lane;
  const bool active = vec < a.vecs;
  const int64_t col = static_cast<int64_t>(active ? vec : 0) * kN;
  const int count = static_cast<int>(std::min<int64_t>(a.chunk, a.n - first));

  const uint32_t none = static_cast<uint32_t>(a.vocab);
  const uint32_t my_key = lane < count ? a.keys[first + lane] : none;
  const uint32_t my_row = lane < count ? a.order[first + lane] : 0u;
  const uint32_t before = first > 0 ? a.keys[first - 1] : none;
  const uint32_t after = first + count < a.n ? a.keys[first + count] : none;

  float acc[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) acc[i] = 0.0f;
  uint32_t key = __builtin_amdgcn_readlane(my_key, 0);
  bool open = key == before;  // the token began in an earlier chunk

  auto flush = [&](uint32_t k, bool began_before, bool goes_on) {
    if (!active) return;
    if (began_before || goes_on) {
      float* to = a.partial + (chunk * 2 + (began_before ? 0 : 1)) * a.dim + col;
#pragma unroll
      for (int i = 0; i < kN; ++i) to[i] = acc[i];
    } else {
      P p;
#pragma unroll
      for (int i = 0; i < kN; ++i) p.v[i] = narrow<T>(acc[i] * a.scale);
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
          if (key != none) flush(key, open, false);
          key = k;
          open = false;
#pragma unroll
          for (int i = 0; i < kN; ++i) acc[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kN; ++i) acc[i] += widen(row[u].v[i]);
      }
    }
  }
  if (key != none) flush(key, open, key == after);
}

// A workgroup per chunk and slice of 256 columns: if a token begins in the chunk and goes on behind it, its partial sums.
constexpr int kJoinThreads = 256;

template <typename T>
__global__ __launch_bounds__(kJoinThreads) void embedding_join_kernel(SumArgs a) {
  const int64_t chunk = blockIdx.x;
  const int64_t first = chunk * a.chunk, next = first + a.chunk;
  if (next >= a.n) return;
  const uint32_t key = a.keys[next - 1];
  if (key == static_cast<uint32_t>(a.vocab) || a.keys[next] != key) return;
  if (first > 0 && a.keys[first] == key && a.keys[first - 1] == key) return;  // it began earlier
  int64_t lo = next, hi = a.n;  // the first entry behind the token's last
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (a.keys[mid] <= key) lo = mid + 1;
    else hi = mid;
  }
  const int64_t last = (lo - 1) / a.chunk;
  const int64_t col = static_cast<int64_t>(blockIdx.y) * kJoinThreads + threadIdx.x;
  if (col >= a.dim) return;
  float acc = a.partial[(chunk * 2 + 1) * a.dim + col];
#pragma unroll 8
  for (int64_t c = chunk + 1; c <= last; ++c) acc += a.partial[c * 2 * a.dim + col];
  static_cast<T*>(a.dweight)[static_cast<int64_t>(key) * a.dim + col] = narrow<T>(acc * a.scale);
}

// ---------------------------------------------------------------- host

constexpr int64_t kMostTokens = int64_t(1) << 28;  // the sums' launch stays below 2^32 lanes

int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }

int chunk_of(int64_t n) { return n <= 16384 ? 16 : n <= 65536 ? 32 : 64; }

void check_shape(int64_t n, int64_t vocab, int64_t dim, int dtype) {
  require(operator_dtype(dtype), "embedding: the dtype must be float32, float16 or bfloat16");
  require(n >= 0 && n <= kMostTokens, "embedding: 0 to 2^28 tokens");
  require(vocab >= 1 && vocab < (int64_t(1) << 31), "embedding: a vocabulary of 1 to 2^31 - 1 rows");
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

struct Workspace {  // of the gradient
  int64_t keys[2], order[2], partial, bytes;
};

Workspace workspace_of(int64_t n, int64_t dim) {
  Workspace w{};
  auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  const int sides = n > kTile ? 2 : 1;
  for (int i = 0; i < sides; ++i) {
    w.keys[i] = take(n * 4);
    w.order[i] = take(n * 4);
  }
  const int64_t chunks = (n + chunk_of(n) - 1) / chunk_of(n);
  w.partial = take(chunks > 1 ? chunks * 2 * dim * 4 : 0);
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
    const int rows = kLookupThreads >> a.log_lanes;
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
    bytes = workspace_of(n, dim).bytes;
  });
  return bytes;
}

int tdm_k5_embedding_grad(const void* grad, const void* tokens, int index_dtype, void* dweight, void* workspace, int64_t workspace_bytes,
                          int64_t n, int64_t vocab, int64_t dim, int dtype, float scale, int64_t padding, tdm_stream stream) {
  return guard([&] {
    check_shape(n, vocab, dim, dtype);
    check_index(index_dtype);
    require(dweight != nullptr && (n == 0 || (grad != nullptr && tokens != nullptr)), "embedding_grad: null pointer");
    const Workspace ws = workspace_of(n, dim);
    require(n == 0 || (workspace != nullptr && workspace_bytes >= ws.bytes), "embedding_grad: the workspace is smaller than tdm_k5_embedding_grad_workspace says");
    require(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "embedding_grad: the workspace must start on 16 bytes");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char* const base = static_cast<char*>(workspace);
    const int es = dtype == TDM_F32 ? 4 : 2;

    SortArgs s{};
    s.tokens = tokens;
    s.zero = dweight;
    s.zero_bytes = vocab * dim * es;
    s.n = n;
    s.vocab = vocab;
    s.padding = padding;
    s.tiles = static_cast<int>(tiles_of(n));
    if (n > 0) {
      s.keys = reinterpret_cast<uint32_t*>(base + ws.keys[0]);
      s.order = reinterpret_cast<uint32_t*>(base + ws.order[0]);
    }
    int bits = 1;
    while ((vocab >> bits) != 0) ++bits;  // keys are 0..vocab
    s.passes = (bits + kDigitBits - 1) / kDigitBits;
    s.digit_bits = (bits + s.passes - 1) / s.passes;
    const int64_t fill = std::min<int64_t>((s.zero_bytes + 65535) / 65536, 2048);
    const dim3 grid(static_cast<unsigned>(s.tiles + fill));
    if (index_dtype == TDM_I64) hipLaunchKernelGGL((embedding_sort_kernel<int64_t>), grid, dim3(kSortThreads), 0, st, s);
    else hipLaunchKernelGGL((embedding_sort_kernel<int32_t>), grid, dim3(kSortThreads), 0, st, s);
    check_launch("embedding_sort launch");
    if (n == 0) return;

    int side = 0;
    for (int64_t run = kTile; run < n; run *= kMergeWays) {
      MergeArgs m{reinterpret_cast<uint32_t*>(base + ws.keys[side]), reinterpret_cast<uint32_t*>(base + ws.order[side]),
                  reinterpret_cast<uint32_t*>(base + ws.keys[side ^ 1]), reinterpret_cast<uint32_t*>(base + ws.order[side ^ 1]), n, run};
      hipLaunchKernelGGL(embedding_merge_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, st, m);
      check_launch("embedding_merge launch");
      side ^= 1;
    }

    const int width = access_width(reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(dweight) | static_cast<uintptr_t>(dim * es), es);
    SumArgs a{};
    a.grad = grad;
    a.keys = reinterpret_cast<uint32_t*>(base + ws.keys[side]);
    a.order = reinterpret_cast<uint32_t*>(base + ws.order[side]);
    a.dweight = dweight;
    a.partial = reinterpret_cast<float*>(base + ws.partial);
    a.n = n;
    a.vocab = vocab;
    a.dim = dim;
    a.chunk = chunk_of(n);
    a.vecs = static_cast<int>(dim * es / width);
    a.slices = (a.vecs + kWave - 1) / kWave;
    a.scale = scale;
    const int64_t chunks = (n + a.chunk - 1) / a.chunk;
    const int64_t groups = (chunks * a.slices + kSumWaves - 1) / kSumWaves;
    require(groups <= (int64_t(1) << 24), "embedding_grad: more than 2^26 chunks and slices");
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      with_width(width, [&](auto w) {
        if constexpr (w.value >= static_cast<int>(sizeof(T)))
          hipLaunchKernelGGL((embedding_sum_kernel<T, w.value>), dim3(static_cast<unsigned>(groups)), dim3(kSumWaves * kWave), 0, st, a);
      });
      check_launch("embedding_sum launch");
      if (chunks > 1) {
        hipLaunchKernelGGL((embedding_join_kernel<T>), dim3(static_cast<unsigned>(chunks), static_cast<unsigned>((dim + kJoinThreads - 1) / kJoinThreads)),
                           dim3(kJoinThreads), 0, st, a);
        check_launch("embedding_join launch");
      }
    });
  });
}

}  // extern "C"
