// K7: the distillation loss from a teacher's top logits, and its gradient.
//
// For a row x of vocab logits, the teacher's k logits t at the columns j_k, the temperature T, the weight a and the target y:
//
//   p = softmax(t / T) over the k entries,   q_T = softmax(x / T),   q_1 = softmax(x)
//   row = a T^2 sum_k p_k (log p_k - log q_T[j_k]) + (1 - a) (-log q_1[y])
//   d row / d x_j = a T (q_T[j] - sum of the p_k with j_k = j) + (1 - a) (q_1[j] - [j = y])
//
// and the loss is the sum or the mean of the rows that count. Loss and gradient come from one visit to the row: the maximum and the
// sums of exponentials need all of it before the first gradient element is known.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/tandem_hip.h"
#include "common.h"
#include "ops_device.h"

namespace tandem_hip {
namespace ops {

namespace {

constexpr int kMostEntries = 1024;  // of the teacher, per row
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct DistillArgs {
  const void* logits;
  const void *index, *teacher, *targets;
  float* rows_loss;        // [rows]
  void* grad;              // null: not wanted
  const float* upstream;   // null: ones
  const float* count;      // rows that count, the mean's divisor; null: counted by the workgroup itself, or `divisor`
  int64_t rows, vocab, ignore;
  int k, index_i64, teacher_dtype, targets_i64;
  int upstream_step;       // 0: one value for all rows
  int counts;              // every workgroup counts the rows itself
  int keep_ones;           // where the upstream value is 1, the gradient there already is right
  float temperature, weight, scale, divisor;
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float ln_of(float x) { return __builtin_amdgcn_logf(x) * kLn2; }

__device__ __forceinline__ float teacher_logit(const DistillArgs& a, int64_t at) {
  if (a.teacher_dtype == TDM_F32) return static_cast<const float*>(a.teacher)[at];
  if (a.teacher_dtype == TDM_F16) return static_cast<float>(static_cast<const _Float16*>(a.teacher)[at]);
  return static_cast<float>(static_cast<const __bf16*>(a.teacher)[at]);
}

__device__ __forceinline__ int64_t index_of(const void* p, int i64, int64_t at) {
  return i64 ? static_cast<const int64_t*>(p)[at] : static_cast<int64_t>(static_cast<const int32_t*>(p)[at]);
}

// Where a row's whole vectors lie: `head` elements before them, `tail` behind. They begin at a multiple of kAlign, 16 or more: rows of an odd
// width touch fewer lines twice then (1031 rows of 50021 fp16 logits 58.7 us, with 16 60.0; 4096 of 32003 bf16 108 to 116, with 16
// 119 to 123). The gradient's row lies at the same distance from 16 bytes.
struct Body {
  int head, vecs, tail;
};
template <int kAlign, typename T>
__device__ __forceinline__ Body body_of(const T* x, int64_t vocab) {
  constexpr int kN = 16 / static_cast<int>(sizeof(T));
  const int head = static_cast<int>(std::min<int64_t>(vocab, ((kAlign - (reinterpret_cast<uintptr_t>(x) & (kAlign - 1))) & (kAlign - 1)) / sizeof(T)));
  const int vecs = static_cast<int>((vocab - head) / kN);
  return Body{head, vecs, static_cast<int>(vocab - head - static_cast<int64_t>(vecs) * kN)};
}

// A running maximum m and the sums of exp2(c (x - m)) (and at log2(e) for the target's share). Where nothing but -inf has been seen the
// sums are zero and m is -inf; `base` is what stands in for m then. The difference comes first: c x would overflow for masks of the type's
// lowest value.
__device__ __forceinline__ float base_of(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// What the two temperatures, T and 1, need of d = x - m: kOne exponential where one of them does for both parts (a = 0, a = 1 or T = 1);
// kTwo; or one again, F, of which both are powers, for T = 2 (F, F^2) and T = 1.5 (F^2, F^3): 1031 rows of 50021 fp16
// logits take 57 us instead of 64, 4096 rows 196 and 201 instead of 212. Every other temperature takes two.
enum Mix { kOne, kTwo, kSquare, kCube };
Mix mix_of(float weight, float temperature) {
  if (weight <= 0.0f || weight >= 1.0f || temperature == 1.0f) return kOne;
  return temperature == 2.0f ? kSquare : temperature == 1.5f ? kCube : kTwo;
}
// What d is multiplied with in F's exponent: log2(e) / T, of kCube log2(e) / 3.
template <Mix kMix>
__device__ __forceinline__ float rate_of(const DistillArgs& a) {
  return kMix == kCube ? kLog2e / 3.0f : a.weight > 0.0f ? kLog2e / a.temperature : kLog2e;
}
template <Mix kMix>
struct Powers {  // soft = exp(d / T), hard = exp(d)
  float f, other = 0.0f;
  __device__ __forceinline__ Powers(float d, float c) : f(exp2_of(d * c)) {
    if (kMix == kTwo) other = exp2_of(d * kLog2e);
  }
  __device__ __forceinline__ float soft() const { return kMix == kCube ? f * f : f; }
  __device__ __forceinline__ float hard() const { return kMix == kOne ? f : kMix == kTwo ? other : soft() * f; }
  __device__ __forceinline__ float add_hard(float to) const { return kMix == kOne ? 0.0f : kMix == kTwo ? to + other : fmaf(soft(), f, to); }
  __device__ __forceinline__ float weighed(float of_soft, float of_hard) const {
    return kMix == kOne ? of_soft * f : kMix == kTwo ? fmaf(of_hard, other, of_soft * f) : soft() * fmaf(of_hard, f, of_soft);
  }
};

template <Mix kMix>
struct Sums {
  float m = -__builtin_inff(), z = 0.0f, z1 = 0.0f;

  template <int kN>
  __device__ __forceinline__ void take(const float (&f)[kN], float c) {
    float top = f[0];
#pragma unroll
    for (int i = 1; i < kN; ++i) top = fmaxf(top, f[i]);
    top = fmaxf(top, m);
    const float base = base_of(top);
    float s = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const Powers<kMix> e(f[i] - base, c);
      s += e.soft();
      s1 = e.add_hard(s1);
    }
    const Powers<kMix> e(m - base, c);
    z = fmaf(z, e.soft(), s);
    if (kMix != kOne) z1 = fmaf(z1, e.hard(), s1);
    m = top;
  }
  // the same sums with the maximum `top` of several
  __device__ __forceinline__ void lift(float top, float c) {
    const float base = base_of(top);
    const Powers<kMix> e(m - base, c);
    z *= e.soft();
    if (kMix != kOne) z1 *= e.hard();
    m = top;
  }
};

// This wave's part of the number of rows that count, kThreads lanes asking.
template <int kThreads>
__device__ __forceinline__ float counted_by_wave(const DistillArgs& a) {
  float n = 0.0f;
#pragma unroll 16
  for (int64_t r = threadIdx.x; r < a.rows; r += kThreads) n += index_of(a.targets, a.targets_i64, r) != a.ignore ? 1.0f : 0.0f;
  return wave_sum(n);
}

// What a wave knows about a row, for the workgroup's others.
struct WaveRow {
  float m, z, z1, t_m, t_z;
  uint32_t flags;
};
constexpr uint32_t kTwice = 1, kBad = 2;  // a column named twice; something outside the vocabulary, or a NaN of the teacher's

// Over the first kWaves (a power of two, at most 16) lanes of a wave; every lane gets it.
template <int kWaves>
__device__ __forceinline__ float sum_of(float x) {
  if constexpr (kWaves >= 2) x = dpp_step<0x111, 0xf>(x, 0.0f, Add{});
  if constexpr (kWaves >= 4) x = dpp_step<0x112, 0xf>(x, 0.0f, Add{});
  if constexpr (kWaves >= 8) x = dpp_step<0x114, 0xf>(x, 0.0f, Add{});
  if constexpr (kWaves >= 16) x = dpp_step<0x118, 0xf>(x, 0.0f, Add{});
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), kWaves - 1));
}
template <int kWaves>
__device__ __forceinline__ float max_of(float x) {
  const float none = -__builtin_inff();
  if constexpr (kWaves >= 2) x = dpp_step<0x111, 0xf>(x, none, Max{});
  if constexpr (kWaves >= 4) x = dpp_step<0x112, 0xf>(x, none, Max{});
  if constexpr (kWaves >= 8) x = dpp_step<0x114, 0xf>(x, none, Max{});
  if constexpr (kWaves >= 16) x = dpp_step<0x118, 0xf>(x, none, Max{});
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), kWaves - 1));
}

constexpr uint32_t kNoColumn = 0xffffffffu;

// A workgroup of kG lanes per row, and on to the row a grid further. The row is read once into kHeld vectors of every lane's
// registers (kHeld 0: a row that does not fit is read again for its gradient); every lane keeps its own running maximum and sum, so the
// exponentials are taken as the vectors arrive, and one barrier joins the waves. While the gradient of a row is computed, each of
// its vectors makes room for the next row's: loads, exponentials and stores are under way at the same time with one workgroup per
// compute unit. The teacher's entries are one lane's each (k <= kG): their elements and the target's are written again after the row, behind
// a second barrier. Columns named twice are found by a hash table in LDS, and only then summed over all entries. 8192 rows of 131072 bf16
// logits and their gradient take 809 us, 5.3 TB/s: bound by memory, reads and writes mixed (797 us with the exponentials taken out).
template <typename T, int kG, int kHeld, Mix kMix>
__global__ __launch_bounds__(kG, 4) void distill_kernel(DistillArgs a, int log_table) {
  constexpr int kN = per_vec<T>(), kWaves = kG / kWave;
  constexpr int kAlign = sizeof(T) == 4 ? 128 : 64;  // at most 31 + 7 elements outside the vectors: a wave's
  __shared__ WaveRow s_wave[2][kWaves];
  __shared__ float s_part[2][kWaves];
  __shared__ int64_t s_cover[2];
  extern __shared__ uint32_t s_table[];  // 2^log_table columns, then k columns and k values of a row with a column named twice
  uint32_t* const s_col = s_table + (1 << log_table);
  float* const s_val = reinterpret_cast<float*>(s_col + a.k);
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const bool soft = a.weight > 0.0f, hard = a.weight < 1.0f;
  const float inv_t = uniform(1.0f / a.temperature);
  const float c = uniform(rate_of<kMix>(a));

  auto row_at = [&](int64_t row) { return static_cast<const T*>(a.logits) + row * a.vocab; };

  constexpr int kAhead = 4;          // vectors in flight of a row that is read twice, or for its loss alone
  constexpr int kEarly = kHeld / 2;  // vectors of the next row that are read while this row's gradient is written
  Vec16 held[kHeld > 0 ? kHeld : 1];
  Stretch from = stretch(nullptr, 0);
  T edge_held = narrow<T>(0.0f);
  uint32_t col = kNoColumn;  // of the teacher's entry of this lane
  float t = -__builtin_inff();
  bool bad = false;
  const int lane16 = tid * 16;
  auto edge_of = [&](const Body& b) { return tid < b.head ? tid : tid - b.head < b.tail ? b.head + b.vecs * kN + tid - b.head : -1; };
  auto fetch_small = [&](int64_t row, const T* x, const Body& b) {  // the edge, the teacher's entry
    if (wave == 0) {
      const int e = edge_of(b);
      if (e >= 0) edge_held = x[e];
    }
    if (!soft || wave * kWave >= a.k) return;
    col = kNoColumn;
    bad = false;
    t = -__builtin_inff();
    if (tid < a.k) {
      const int64_t j = index_of(a.index, a.index_i64, row * a.k + tid);
      const float logit = teacher_logit(a, row * a.k + tid);
      if (j >= 0) {
        bad = j >= a.vocab || logit != logit;
        if (!bad) {
          col = static_cast<uint32_t>(j);
          t = logit;
        }
      }
    }
  };

  auto write_zeros = [&](T* g) {
    const Body b = body_of<kAlign>(g, a.vocab);
    const Vec16 zero = {0u, 0u, 0u, 0u};
    for (int v = tid; v < b.vecs; v += kG) __builtin_nontemporal_store(zero, reinterpret_cast<Vec16*>(g + b.head) + v);
    const int e = edge_of(b);
    if (e >= 0) g[e] = narrow<T>(0.0f);
  };
  // The first row from `row` on, a grid apart, that there is work for; the rows before it that do not count get their zeros. a.rows: none.
  auto seek = [&](int64_t row) {
    for (; row < a.rows; row += gridDim.x) {
      if (a.keep_ones && a.upstream[row * a.upstream_step] == 1.0f) continue;
      if (a.targets == nullptr || index_of(a.targets, a.targets_i64, row) != a.ignore) return row;
      if (a.rows_loss != nullptr && tid == 0) a.rows_loss[row] = 0.0f;
      if (a.grad != nullptr) write_zeros(static_cast<T*>(a.grad) + row * a.vocab);
    }
    return a.rows;
  };

  for (int i = tid; i < 1 << log_table; i += kG) s_table[i] = kNoColumn;
  if (tid < 2) s_cover[tid] = -1;
  int64_t row = seek(blockIdx.x);
  if (row == a.rows) return;
  Body body = body_of<kAlign>(row_at(row), a.vocab);
  fetch_small(row, row_at(row), body);
  if constexpr (kHeld > 0) {
    from = stretch(row_at(row) + body.head, body.vecs * 16);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = load16(from, lane16, i * kG * 16);
  }
  if (a.counts) {
    const float n = counted_by_wave<kG>(a);
    if (lane == 0) s_part[0][wave] = n;
  }
  __syncthreads();
  const float counted = a.counts ? fmaxf(sum_of<kWaves>(s_part[0][lane % kWaves]), 1.0f) : a.count == nullptr ? a.divisor : *a.count;
  const float scale = uniform(a.scale / counted);
  __syncthreads();  // s_part is the rows' from here on

  for (int turn = 0; row < a.rows; turn ^= 1) {
    const T* const x = row_at(row);
    T* const g = a.grad == nullptr ? nullptr : static_cast<T*>(a.grad) + row * a.vocab;
    const float up = a.upstream == nullptr ? 1.0f : a.upstream[row * a.upstream_step];
    const int64_t y = hard ? index_of(a.targets, a.targets_i64, row) : -1;
    const bool y_bad = hard && (y < 0 || y >= a.vocab);
    const int edge = edge_of(body);
    const float x_col = col != kNoColumn ? widen(x[col]) : 0.0f;
    const float x_y = hard && !y_bad ? widen(x[y]) : 0.0f;
    const float edge_x = edge >= 0 ? widen(edge_held) : -__builtin_inff();

    const int64_t next = seek(row + gridDim.x);
    const T* const nx = row_at(next < a.rows ? next : row);
    const Body next_body = body_of<kAlign>(nx, a.vocab);

    // the row's maximum and sums
    Sums<kMix> sums;
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        if (tid + i * kG < body.vecs) {
          float f[kN];
          unpack16<T>(held[i], f);
          sums.take(f, c);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      const Vec16* const vecs = reinterpret_cast<const Vec16*>(x + body.head);
      for (int v = tid; v < body.vecs; v += kG * kAhead) {
        Vec16 ahead[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (v + u * kG < body.vecs) ahead[u] = vecs[v + u * kG];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (v + u * kG < body.vecs) {
            float f[kN];
            unpack16<T>(ahead[u], f);
            sums.take(f, c);
          }
      }
    }
    {
      const float f[1] = {edge_x};
      sums.take(f, c);
    }
    // the teacher's, and whether a column comes twice
    const float ck = kLog2e * inv_t;
    const bool teaches = soft && wave * kWave < a.k;  // this wave has entries
    uint32_t slot = kNoColumn;
    WaveRow mine;
    mine.t_m = -__builtin_inff();
    mine.t_z = 0.0f;
    mine.flags = 0;
    if (teaches) {
      bool twice = false;
      if (col != kNoColumn) {
        uint32_t at = (col * 2654435761u) >> (32 - log_table);
        for (;;) {
          const uint32_t old = atomicCAS(&s_table[at], kNoColumn, col);
          if (old == kNoColumn) {
            slot = at;
            break;
          }
          if (old == col) {
            twice = true;
            break;
          }
          at = (at + 1) & ((1u << log_table) - 1);
        }
      }
      mine.t_m = wave_max(t);
      mine.t_z = wave_sum(exp2_of((t - base_of(mine.t_m)) * ck));
      mine.flags = (__ballot(twice) != 0 ? kTwice : 0) | (__ballot(bad) != 0 ? kBad : 0);
    }
    mine.m = wave_max(sums.m);
    sums.lift(mine.m, c);
    mine.z = wave_sum(sums.z);
    mine.z1 = kMix != kOne ? wave_sum(sums.z1) : mine.z;
    float m = mine.m, z = mine.z, z1 = mine.z1, t_m = mine.t_m, t_z = mine.t_z;
    bool any_twice = mine.flags & kTwice, any_bad = mine.flags & kBad;
    if constexpr (kWaves > 1) {
      if (lane == 0) s_wave[turn][wave] = mine;
      __syncthreads();
      const WaveRow w = s_wave[turn][lane % kWaves];  // at most 16 waves: every row of 16 lanes has them all, some more than once
      m = max_of<kWaves>(w.m);
      Sums<kMix> part;
      part.m = w.m;
      part.z = w.z;
      part.z1 = w.z1;
      part.lift(m, c);
      z = sum_of<kWaves>(part.z);
      z1 = kMix != kOne ? sum_of<kWaves>(part.z1) : z;
      if (soft) {
        t_m = max_of<kWaves>(w.t_m);
        t_z = sum_of<kWaves>(w.t_z * exp2_of((w.t_m - base_of(t_m)) * ck));
      }
      any_twice = __ballot(w.flags & kTwice) != 0;
      any_bad = __ballot(w.flags & kBad) != 0;
    }
    any_bad = any_bad || y_bad;
    const bool taught = soft && t_m != -__builtin_inff();
    const bool idle = !taught && !hard && !any_bad;  // the teacher says nothing: zeros, whatever the logits are
    // nothing but -inf: the definition has no value
    const float wrong = any_bad || (m == -__builtin_inff() && !idle) ? __builtin_nanf("") : 0.0f;
    const float base = uniform(base_of(m));

    // the loss
    float p = 0.0f;
    if (teaches || wave == 0) {
      float part = 0.0f;
      if (taught && col != kNoColumn) {
        const float tk = (t - t_m) * inv_t;
        p = exp2_of(tk * kLog2e) / t_z;
        if (!(p == 0.0f)) part = a.weight * a.temperature * a.temperature * p * (tk - ln_of(t_z) - ((x_col - base) * inv_t - ln_of(z)));
      }
      if (hard && tid == 0) part += (1.0f - a.weight) * (ln_of(z1) - (x_y - base));
      part = wave_sum(part);
      if (lane == 0) s_part[turn][wave] = part;
      if (slot != kNoColumn) s_table[slot] = kNoColumn;
      if (any_twice && tid < a.k) {
        s_col[tid] = col;
        s_val[tid] = p;
      }
      if (taught && hard && col != kNoColumn && col == static_cast<uint32_t>(y)) s_cover[turn] = row;
    }

    // the gradient: from the sums, then the teacher's columns and the target again, with what they take off
    const float s = scale * up + wrong;
    const float w_t = uniform(taught ? s * a.weight * a.temperature : wrong), w_1 = uniform(hard ? s * (1.0f - a.weight) : 0.0f);
    const float k_t = uniform((kMix != kOne ? w_t : w_t + w_1) * __builtin_amdgcn_rcpf(z)), k_1 = kMix != kOne ? uniform(w_1 * __builtin_amdgcn_rcpf(z1)) : 0.0f;
    auto slope = [&](float f) {
      return Powers<kMix>(f - base, c).weighed(k_t, k_1);
    };
    if (g != nullptr && edge >= 0) g[edge] = narrow<T>(idle ? 0.0f : slope(edge_x) + wrong);
    if (g != nullptr && idle) write_zeros(g);
    const uint32_t my_col = col;
    if (next < a.rows) fetch_small(next, nx, next_body);
    // 16-bit gradients: one multiply-add and the exponential, the row's maximum in the exponent, and where every exponential has a factor of its
    // own that too, its sign apart. That is off by 2^-24 of the exponent's terms: far less than the store's rounding while they
    // stay below 1024. Other rows, and what does not fit the registers, are read again.
    constexpr bool kApart = kMix == kOne || kMix == kTwo;
    const float off = uniform((kApart ? __builtin_amdgcn_logf(fabsf(k_t)) : 0.0f) - base * c);
    const float off1 = kMix == kTwo ? uniform(__builtin_amdgcn_logf(fabsf(k_1)) - base * kLog2e) : 0.0f;
    const uint32_t sign = kApart && s < 0.0f ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
    const bool held_fits = sizeof(T) == 4 || (fabsf(base * c) < 1024.0f && (kMix != kTwo || fabsf(base * kLog2e) < 1024.0f));
    if constexpr (kHeld > 0) {
      from = stretch(nx + next_body.head, next < a.rows ? next_body.vecs * 16 : 0);
      const Stretch to = stretch(g + body.head, g != nullptr && !idle && held_fits ? body.vecs * 16 : 0);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        if (g != nullptr) {
          asm("" : "+v"(held[i]));  // unpacked anew: the floats of the sums, kept, would take twice the registers
          float f[kN];
          unpack16<T>(held[i], f);
#pragma unroll
          for (int e = 0; e < kN; ++e) {
            if constexpr (sizeof(T) == 4) f[e] = slope(f[e]);
            else if constexpr (kApart) f[e] = exp2_of(fmaf(f[e], c, off)) + (kMix == kTwo ? exp2_of(fmaf(f[e], kLog2e, off1)) : 0.0f);
            else {
              const float p = exp2_of(fmaf(f[e], c, off));
              f[e] = (kMix == kCube ? p * p : p) * fmaf(k_1, p, k_t);
            }
          }
          Vec16 out = pack16<T>(f);
          if constexpr (sizeof(T) == 2 && kApart) out ^= sign;
          store16(out, to, lane16, i * kG * 16);
        }
        if (i < kEarly) held[i] = load16(from, lane16, i * kG * 16);
        __builtin_amdgcn_sched_barrier(0);  // one vector at a time: interleaved, they take twice the registers
      }
    }
    if (g != nullptr && !idle && (kHeld == 0 || !held_fits)) {
      for (int v = tid; v < body.vecs; v += kG) {
        float f[kN];
        unpack16<T>(reinterpret_cast<const Vec16*>(x + body.head)[v], f);
#pragma unroll
        for (int e = 0; e < kN; ++e) f[e] = slope(f[e]);
        reinterpret_cast<Vec16*>(g + body.head)[v] = pack16<T>(f);
      }
    }
    __syncthreads();
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int i = kEarly; i < kHeld; ++i) held[i] = load16(from, lane16, i * kG * 16);
    }
    if (a.rows_loss != nullptr && tid == 0) {
      float loss = wrong;
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        if (w == 0 || (soft && w * kWave < a.k)) loss += s_part[turn][w];
      a.rows_loss[row] = loss;
    }
    if (g != nullptr && !any_bad) {
      if (taught && my_col != kNoColumn) {
        float down = w_t * p;  // all that falls on this column: an entry named twice comes out the same for each
        if (any_twice) {
          down = 0.0f;
          for (int e = 0; e < a.k; ++e) down += s_col[e] == my_col ? w_t * s_val[e] : 0.0f;
        }
        if (hard && my_col == static_cast<uint32_t>(y)) down += w_1;
        g[my_col] = narrow<T>(slope(x_col) - down);
      }
      if (hard && tid == 0 && s_cover[turn] != row) g[y] = narrow<T>(slope(x_y) - w_1);
    }
    row = next;
    body = next_body;
  }
}

// Short rows: 16 lanes a row, so that what a row needs once is done for four rows by every instruction of a wave (8192 rows of 256
// floats, 16 entries, two temperatures: 11.2 us; 14.1 with a wave a row). kHeld vectors of the row and kEntries of the teacher's entries per lane.
constexpr int kShortLanes = 16, kShortThreads = 256, kShortRows = kShortThreads / kShortLanes;

template <typename T, int kHeld, int kEntries, Mix kMix>
__global__ __launch_bounds__(kShortThreads) void distill_short_kernel(DistillArgs a) {
  constexpr int kN = per_vec<T>();
  extern __shared__ uint32_t s_short[];  // k columns and k values of every row
  const int sub = threadIdx.x % kShortLanes, place = threadIdx.x / kShortLanes;
  __shared__ float s_count[kShortThreads / kWave];
  uint32_t* const s_col = s_short + place * 2 * a.k;
  float* const s_val = reinterpret_cast<float*>(s_col + a.k);
  const bool soft = a.weight > 0.0f, hard = a.weight < 1.0f;
  const float inv_t = 1.0f / a.temperature, ck = kLog2e * inv_t, c = rate_of<kMix>(a);
  const float lowest = -__builtin_inff();

  const int64_t asked = static_cast<int64_t>(blockIdx.x) * kShortRows + place, row = std::min(asked, a.rows - 1);
  const float up = a.upstream == nullptr ? 1.0f : a.upstream[row * a.upstream_step];
  const int64_t y = a.targets == nullptr ? 0 : index_of(a.targets, a.targets_i64, row);
  const bool skip = asked >= a.rows || (a.keep_ones && up == 1.0f), counted = a.targets == nullptr || y != a.ignore, live = !skip && counted;
  const T* const x = static_cast<const T*>(a.logits) + row * a.vocab;
  T* const g = static_cast<T*>(a.grad) + row * a.vocab;  // used where a.grad is given
  const Body body = body_of<16>(x, a.vocab);
  const int edge = sub < body.head ? sub : sub - body.head < body.tail ? body.head + body.vecs * kN + sub - body.head : -1;

  Vec16 held[kHeld];
  float edge_x = lowest;
  if (live) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (sub + i * kShortLanes < body.vecs) held[i] = reinterpret_cast<const Vec16*>(x + body.head)[sub + i * kShortLanes];
    if (edge >= 0) edge_x = widen(x[edge]);
  }
  if (a.counts) {
    const float n = counted_by_wave<kShortThreads>(a);
    if (threadIdx.x % kWave == 0) s_count[threadIdx.x / kWave] = n;
  }
  uint32_t col[kEntries];
  float t[kEntries], x_col[kEntries], t_top = lowest, flags = 0.0f;
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    col[i] = kNoColumn;
    t[i] = lowest;
    x_col[i] = 0.0f;
    const int e = sub + i * kShortLanes;
    if (!live || !soft || e >= a.k) continue;
    const int64_t j = index_of(a.index, a.index_i64, row * a.k + e);
    const float logit = teacher_logit(a, row * a.k + e);
    if (j < 0) continue;
    if (j >= a.vocab || logit != logit) {
      flags = 1.0f;
      continue;
    }
    col[i] = static_cast<uint32_t>(j);
    t[i] = logit;
    x_col[i] = widen(x[j]);
    t_top = fmaxf(t_top, logit);
  }
  if (live && hard && (y < 0 || y >= a.vocab)) flags = 1.0f;
  const bool bad = all_16(flags, Max{}) != 0.0f;
  const float x_y = live && hard && !bad && sub == 0 ? widen(x[y]) : 0.0f;

  Sums<kMix> sums;
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (live && sub + i * kShortLanes < body.vecs) {
      float f[kN];
      unpack16<T>(held[i], f);
      sums.take(f, c);
    }
  {
    const float f[1] = {edge_x};
    sums.take(f, c);
  }
  const float m = all_16(sums.m, Max{}), base = base_of(m);
  sums.lift(m, c);
  const float z = all_16(sums.z, Add{}), z1 = kMix != kOne ? all_16(sums.z1, Add{}) : z;
  const float t_m = all_16(t_top, Max{});
  float t_sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kEntries; ++i) t_sum += exp2_of((t[i] - base_of(t_m)) * ck);
  const float t_z = all_16(t_sum, Add{});
  const bool taught = soft && t_m != lowest, idle = !taught && !hard && !bad;
  const float wrong = bad || (m == lowest && !idle) ? __builtin_nanf("") : 0.0f;

  float p[kEntries], part = 0.0f;
  bool mine = false;  // one of this lane's columns is the target
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    p[i] = 0.0f;
    if (taught && col[i] != kNoColumn) {
      const float tk = (t[i] - t_m) * inv_t;
      p[i] = exp2_of(tk * kLog2e) / t_z;
      if (!(p[i] == 0.0f)) part += a.weight * a.temperature * a.temperature * p[i] * (tk - ln_of(t_z) - ((x_col[i] - base) * inv_t - ln_of(z)));
      mine = mine || (hard && col[i] == static_cast<uint32_t>(y));
    }
    const int e = sub + i * kShortLanes;
    if (e < a.k) {
      s_col[e] = col[i];
      s_val[e] = p[i];
    }
  }
  if (hard && sub == 0) part += (1.0f - a.weight) * (ln_of(z1) - (x_y - base));
  part = all_16(part, Add{});
  const bool covered = all_16(mine ? 1.0f : 0.0f, Max{}) != 0.0f;
  if (a.rows_loss != nullptr && !skip && sub == 0) a.rows_loss[row] = counted ? part + wrong : 0.0f;
  __syncthreads();
  if (a.grad == nullptr || skip) return;

  float count = a.divisor;
  if (a.counts) {
    count = 0.0f;
#pragma unroll
    for (int w = 0; w < kShortThreads / kWave; ++w) count += s_count[w];
    count = fmaxf(count, 1.0f);
  } else if (a.count != nullptr) {
    count = *a.count;
  }
  const float s = a.scale / count * up + wrong;
  const float w_t = taught ? s * a.weight * a.temperature : wrong, w_1 = hard ? s * (1.0f - a.weight) : 0.0f;
  const float k_t = (kMix != kOne ? w_t : w_t + w_1) * __builtin_amdgcn_rcpf(z), k_1 = kMix != kOne ? w_1 * __builtin_amdgcn_rcpf(z1) : 0.0f;
  const bool zeros = !counted || idle;
  auto slope = [&](float f) {
    return Powers<kMix>(f - base, c).weighed(k_t, k_1);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (sub + i * kShortLanes < body.vecs) {
      Vec16 out = {0u, 0u, 0u, 0u};
      if (!zeros) {
        float f[kN];
        unpack16<T>(held[i], f);
#pragma unroll
        for (int e = 0; e < kN; ++e) f[e] = slope(f[e]);
        out = pack16<T>(f);
      }
      reinterpret_cast<Vec16*>(g + body.head)[sub + i * kShortLanes] = out;
    }
  if (edge >= 0) g[edge] = narrow<T>(zeros ? 0.0f : slope(edge_x) + wrong);
  if (zeros || bad) return;
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {  // after the whole vectors, by the same wave
    if (!taught || col[i] == kNoColumn) continue;
    float down = 0.0f;
    for (int e = 0; e < a.k; ++e) down += s_col[e] == col[i] ? w_t * s_val[e] : 0.0f;
    if (hard && col[i] == static_cast<uint32_t>(y)) down += w_1;
    g[col[i]] = narrow<T>(slope(x_col[i]) - down);
  }
  if (hard && sub == 0 && !covered) g[y] = narrow<T>(slope(x_y) - w_1);
}

constexpr int kFoldThreads = 1024;

// Of the waves' values (the same in all of a wave's lanes); every lane gets it.
__device__ __forceinline__ float block_total(float of_wave) {
  __shared__ float s[kFoldThreads / kWave];
  __syncthreads();
  if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = of_wave;
  __syncthreads();
  return sum_of<kFoldThreads / kWave>(s[threadIdx.x % (kFoldThreads / kWave)]);
}

// How many rows count (at least one: a batch without any has loss 0).
__global__ __launch_bounds__(kFoldThreads) void distill_count_kernel(DistillArgs a, float* count) {
  const float n = block_total(counted_by_wave<kFoldThreads>(a));
  if (threadIdx.x == 0) *count = fmaxf(n, 1.0f);
}

__global__ __launch_bounds__(kFoldThreads) void distill_sum_kernel(DistillArgs a, float* loss) {
  float x = 0.0f;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < a.rows; r += kFoldThreads) x += a.rows_loss[r];
  x = block_total(wave_sum(x));
  const float n = a.counts ? fmaxf(block_total(counted_by_wave<kFoldThreads>(a)), 1.0f) : a.count == nullptr ? a.divisor : *a.count;
  if (threadIdx.x == 0) *loss = x / n;
}

// The loss alone of a few long rows: with a workgroup per row most compute units are idle (4 rows of 131072 bf16 logits: 14.2 us and the
// sum's launch; split, 3.6 and 3.6). Every row is split over `slices` workgroups, which leave their maximum and sums; one more workgroup joins them, a wave
// per row, with the teacher's share.
constexpr int kSliceThreads = 256, kMostSlices = kWave;

template <typename T, Mix kMix>
__global__ __launch_bounds__(kSliceThreads) void distill_slice_kernel(DistillArgs a, int slices, int per_slice, WaveRow* parts) {
  constexpr int kN = per_vec<T>(), kWaves = kSliceThreads / kWave, kAhead = 4;
  __shared__ WaveRow s_wave[kWaves];
  const int64_t row = blockIdx.x / slices;
  const int slice = blockIdx.x % slices, tid = threadIdx.x;
  if (a.targets != nullptr && index_of(a.targets, a.targets_i64, row) == a.ignore) return;
  const T* const x = static_cast<const T*>(a.logits) + row * a.vocab;
  const Body body = body_of<16>(x, a.vocab);
  const float c = rate_of<kMix>(a);
  Sums<kMix> sums;
  if (slice == 0) {
    const int edge = tid < body.head ? tid : tid - body.head < body.tail ? body.head + body.vecs * kN + tid - body.head : -1;
    const float f[1] = {edge >= 0 ? widen(x[edge]) : -__builtin_inff()};
    sums.take(f, c);
  }
  const Vec16* const from = reinterpret_cast<const Vec16*>(x + body.head);
  const int end = std::min((slice + 1) * per_slice, body.vecs);
  for (int v = slice * per_slice + tid; v < end; v += kSliceThreads * kAhead) {
    Vec16 held[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (v + u * kSliceThreads < end) held[u] = from[v + u * kSliceThreads];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (v + u * kSliceThreads < end) {
        float f[kN];
        unpack16<T>(held[u], f);
        sums.take(f, c);
      }
  }
  WaveRow mine{};
  mine.m = wave_max(sums.m);
  sums.lift(mine.m, c);
  mine.z = wave_sum(sums.z);
  mine.z1 = kMix != kOne ? wave_sum(sums.z1) : mine.z;
  if (tid % kWave == 0) s_wave[tid / kWave] = mine;
  __syncthreads();
  if (tid >= kWave) return;
  const WaveRow w = s_wave[tid % kWaves];
  Sums<kMix> part;
  part.m = w.m;
  part.z = w.z;
  part.z1 = w.z1;
  WaveRow all{};
  all.m = max_of<kWaves>(w.m);
  part.lift(all.m, c);
  all.z = sum_of<kWaves>(part.z);
  all.z1 = kMix != kOne ? sum_of<kWaves>(part.z1) : all.z;
  if (tid == 0) parts[blockIdx.x] = all;
}

template <typename T, Mix kMix>
__global__ __launch_bounds__(kFoldThreads) void distill_slices_loss_kernel(DistillArgs a, int slices, const WaveRow* parts, float* loss, int each_row) {
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const bool soft = a.weight > 0.0f, hard = a.weight < 1.0f;
  const float lowest = -__builtin_inff(), inv_t = 1.0f / a.temperature, ck = kLog2e * inv_t, c = rate_of<kMix>(a);
  float total = 0.0f, count = 0.0f;
  for (int64_t row = wave; row < a.rows; row += kFoldThreads / kWave) {
    const int64_t y = a.targets == nullptr ? 0 : index_of(a.targets, a.targets_i64, row);
    if (a.targets != nullptr && y == a.ignore) {
      if (each_row && lane == 0) loss[row] = 0.0f;
      continue;
    }
    const T* const x = static_cast<const T*>(a.logits) + row * a.vocab;
    WaveRow w{};
    if (lane < slices) w = parts[row * slices + lane];
    else w.m = lowest;
    Sums<kMix> part;
    part.m = w.m;
    part.z = w.z;
    part.z1 = w.z1;
    const float m = wave_max(w.m), base = base_of(m);
    part.lift(m, c);
    const float z = wave_sum(part.z), z1 = kMix != kOne ? wave_sum(part.z1) : z;
    bool bad = hard && (y < 0 || y >= a.vocab);
    auto entry = [&](int e, float& t) {  // its column, or -1
      const int64_t j = index_of(a.index, a.index_i64, row * a.k + e);
      t = teacher_logit(a, row * a.k + e);
      if (j < 0) return int64_t(-1);
      if (j < a.vocab && t == t) return j;
      bad = true;
      return int64_t(-1);
    };
    float t, t_top = lowest, t_sum = 0.0f, term = 0.0f;
    for (int e = lane; soft && e < a.k; e += kWave)
      if (entry(e, t) >= 0) t_top = fmaxf(t_top, t);
    const float t_m = wave_max(t_top);
    const bool taught = soft && t_m != lowest;
    if (taught) {
      for (int e = lane; e < a.k; e += kWave)
        if (entry(e, t) >= 0) t_sum += exp2_of((t - t_m) * ck);
      const float t_z = wave_sum(t_sum);
      for (int e = lane; e < a.k; e += kWave) {
        const int64_t j = entry(e, t);
        const float tk = (t - t_m) * inv_t, p = j >= 0 ? exp2_of(tk * kLog2e) / t_z : 0.0f;
        if (!(p == 0.0f)) term += a.weight * a.temperature * a.temperature * p * (tk - ln_of(t_z) - ((widen(x[j]) - base) * inv_t - ln_of(z)));
      }
    }
    bad = __ballot(bad) != 0;
    if (hard && !bad && lane == 0) term += (1.0f - a.weight) * (ln_of(z1) - (widen(x[y]) - base));
    const bool idle = !taught && !hard && !bad;
    const float row_loss = wave_sum(term) + (bad || (m == lowest && !idle) ? __builtin_nanf("") : 0.0f);
    if (each_row && lane == 0) loss[row] = row_loss;
    total += row_loss;
    count += 1.0f;
  }
  if (each_row) return;
  total = block_total(total);
  count = block_total(count);
  if (threadIdx.x == 0) *loss = total / (a.counts ? fmaxf(count, 1.0f) : a.divisor);
}

// ---------------------------------------------------------------- host

void check_how(const tdm_distill_how* h) {
  require(h != nullptr, "distill: null description");
  require(operator_dtype(h->dtype), "distill: the logits must be float32, float16 or bfloat16");
  require(operator_dtype(h->teacher_dtype), "distill: the teacher's logits must be float32, float16 or bfloat16");
  require(h->index_dtype == TDM_I64 || h->index_dtype == TDM_I32, "distill: the teacher's columns must be int64 or int32");
  require(h->target_dtype == TDM_I64 || h->target_dtype == TDM_I32, "distill: the targets must be int64 or int32");
  require(h->rows >= 0 && h->rows <= (int64_t(1) << 24), "distill: 0 to 2^24 rows");  // counted exactly in fp32
  require(h->vocab >= 1 && h->vocab < (int64_t(1) << 31), "distill: 1 to 2^31 - 1 logits in a row");
  require(h->k >= 1 && h->k <= kMostEntries, "distill: 1 to 1024 teacher's logits in a row");
  require(h->temperature > 0.0f && h->temperature < std::numeric_limits<float>::infinity(), "distill: the temperature must be positive and finite");
  require(h->weight >= 0.0f && h->weight <= 1.0f, "distill: the teacher's weight must lie between 0 and 1");
  require(h->reduction == TDM_DISTILL_NONE || h->reduction == TDM_DISTILL_MEAN || h->reduction == TDM_DISTILL_SUM, "distill: unknown reduction");
}

template <class F>
void with_mix(Mix mix, F&& f) {
  switch (mix) {
    case kOne: f(std::integral_constant<Mix, kOne>{}); return;
    case kSquare: f(std::integral_constant<Mix, kSquare>{}); return;
    case kCube: f(std::integral_constant<Mix, kCube>{}); return;
    default: f(std::integral_constant<Mix, kTwo>{}); return;
  }
}

constexpr int64_t kCountBytes = 256;
constexpr int kComputeUnits = 256;

// Rows up to which every workgroup counts the targets itself (64 KiB of them from L2) instead of a launch that does.
constexpr int64_t kCountRows = 8192;
// Rows up to which the loss alone of long rows is split over the rows' length: the joining workgroup has a wave for two of them.
constexpr int64_t kSlicedRows = 32;

int64_t workspace_bytes_of(const tdm_distill_how& h) {
  return kCountBytes + std::max<int64_t>(h.reduction == TDM_DISTILL_NONE ? 0 : h.rows * 4, h.rows <= kSlicedRows ? h.rows * kMostSlices * static_cast<int64_t>(sizeof(WaveRow)) : 0);
}

}  // namespace

}  // namespace ops
}  // namespace tandem_hip

using namespace tandem_hip;
using namespace tandem_hip::ops;

extern "C" {

int64_t tdm_k7_distill_workspace(const tdm_distill_how* how) {
  int64_t bytes = -1;
  guard([&] {
    check_how(how);
    bytes = workspace_bytes_of(*how);
  });
  return bytes;
}

int tdm_k7_distill(const tdm_distill_how* how, const void* logits, const void* teacher_index, const void* teacher_logits, const void* targets,
                   float* loss, void* grad, const float* upstream, int keep_ones, void* workspace, int64_t workspace_bytes, tdm_stream stream) {
  return guard([&] {
    check_how(how);
    const tdm_distill_how& h = *how;
    require(h.rows == 0 || h.weight == 1.0f || targets != nullptr, "distill: a weight below 1 needs targets");
    require(loss != nullptr || grad != nullptr || h.rows == 0, "distill: neither loss nor gradient is wanted");
    require(h.rows == 0 || (logits != nullptr && ((teacher_index != nullptr && teacher_logits != nullptr) || h.weight == 0.0f)), "distill: null pointer");
    require(workspace != nullptr && workspace_bytes >= workspace_bytes_of(h) && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
            "distill: the workspace starts on 16 bytes and holds tdm_k7_distill_workspace bytes");
    require(grad == nullptr || (reinterpret_cast<uintptr_t>(grad) & 15) == (reinterpret_cast<uintptr_t>(logits) & 15),
            "distill: the gradient must start at the logits' distance from a 16-byte boundary");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    float* const count = static_cast<float*>(workspace);
    float* const rows_loss = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCountBytes);
    const bool mean = h.reduction == TDM_DISTILL_MEAN;
    DistillArgs a{};
    a.logits = logits;
    a.index = teacher_index;
    a.teacher = teacher_logits;
    a.targets = targets;
    a.rows_loss = loss == nullptr ? nullptr : h.reduction == TDM_DISTILL_NONE ? loss : rows_loss;
    a.grad = grad;
    a.upstream = upstream;
    a.counts = mean && targets != nullptr;
    a.divisor = mean ? static_cast<float>(std::max<int64_t>(h.rows, 1)) : 1.0f;
    a.rows = h.rows;
    a.vocab = h.vocab;
    a.ignore = h.ignore_index;
    a.k = h.k;
    a.index_i64 = h.index_dtype == TDM_I64;
    a.teacher_dtype = h.teacher_dtype;
    a.targets_i64 = h.target_dtype == TDM_I64;
    a.upstream_step = h.reduction == TDM_DISTILL_NONE ? 1 : 0;
    a.keep_ones = keep_ones != 0 && upstream != nullptr;
    a.temperature = h.temperature;
    a.weight = h.weight;
    a.scale = h.scale;
    const int64_t all_vecs = h.vocab * (h.dtype == TDM_F32 ? 4 : 2) / 16;
    if (grad == nullptr && h.rows > 0 && h.rows <= kSlicedRows && all_vecs > 2048) {
      const int slices = static_cast<int>(std::min<int64_t>(kMostSlices, std::min<int64_t>((all_vecs + 1023) / 1024, 512 / h.rows)));
      const int per_slice = static_cast<int>((all_vecs + slices - 1) / slices);
      WaveRow* const parts = reinterpret_cast<WaveRow*>(rows_loss);
      with_dtype(h.dtype, [&](auto t) {
        using T = decltype(t);
        auto launch = [&](auto m) {
          hipLaunchKernelGGL((distill_slice_kernel<T, m.value>), dim3(static_cast<unsigned>(h.rows * slices)), dim3(kSliceThreads), 0, st, a, slices, per_slice, parts);
          check_launch("distill_slice launch");
          hipLaunchKernelGGL((distill_slices_loss_kernel<T, m.value>), dim3(1), dim3(kFoldThreads), 0, st, a, slices, parts, loss, h.reduction == TDM_DISTILL_NONE);
          check_launch("distill_slices_loss launch");
        };
        with_mix(mix_of(h.weight, h.temperature), launch);
      });
      return;
    }
    // One wave per row where that suffices: what a row needs once (a chain of loads, sums over lanes, logarithms) takes a larger workgroup as
    // long, and fewer rows are under way then. 16384 rows of 3500 fp16 logits: 65 us with one wave, 127 with four; of
    // 8000 logits 2048 rows 20 and 24 us, but 1024 rows 14.5 and 14.4, 512 rows 13.0 and 10.8.
    const bool many = h.rows > 4 * kComputeUnits;
    const bool one_wave = h.k <= 64 && all_vecs > 64 && (all_vecs <= 256 || (many && all_vecs <= (grad == nullptr ? 8192 : 1024)));
    if (a.counts && (h.rows > kCountRows || one_wave)) {  // a workgroup of one wave does not count
      hipLaunchKernelGGL(distill_count_kernel, dim3(1), dim3(kFoldThreads), 0, st, a, count);
      check_launch("distill_count launch");
      a.counts = 0;
      a.count = count;
    }
    if (h.rows > 0) {
      int log_table = 6;  // at most half full
      while ((1 << log_table) < 2 * h.k) ++log_table;
      const unsigned lds = ((1u << log_table) + 2u * h.k) * 4u;
      with_dtype(h.dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t vecs = h.vocab * static_cast<int64_t>(sizeof(T)) / 16;
        auto launch = [&](auto g, auto held, auto m) {
          // about as many workgroups as the GPU holds at once: they go on to further rows
          const int64_t grid = std::min<int64_t>(h.rows, kComputeUnits * (held.value == 0 || g.value == 64 ? 2048 : 1024) / g.value);
          hipLaunchKernelGGL((distill_kernel<T, g.value, held.value, m.value>), dim3(static_cast<unsigned>(grid)), dim3(g.value), lds, st, a, log_table);
        };
        auto pick = [&](auto m) {
          using std::integral_constant;
          const integral_constant<int, 64> g64{};
          const integral_constant<int, 128> g128{};
          const integral_constant<int, 256> g256{};
          const integral_constant<int, 512> g512{};
          const integral_constant<int, 1024> g1024{};
          auto launch_short = [&](auto held, auto entries) {
            const unsigned bytes = static_cast<unsigned>(kShortRows * h.k * 8);
            hipLaunchKernelGGL((distill_short_kernel<T, held.value, entries.value, m.value>), dim3(static_cast<unsigned>((h.rows + kShortRows - 1) / kShortRows)),
                               dim3(kShortThreads), bytes, st, a);
          };
          if (h.k <= 16 && vecs <= 32) launch_short(integral_constant<int, 2>{}, integral_constant<int, 1>{});
          else if (h.k <= 16 && vecs <= 64) launch_short(integral_constant<int, 4>{}, integral_constant<int, 1>{});
          else if (h.k <= 64 && vecs <= 64) launch_short(integral_constant<int, 4>{}, integral_constant<int, 4>{});
          else if (one_wave && vecs <= 256) launch(g64, integral_constant<int, 4>{}, m);
          else if (one_wave && vecs <= 512) launch(g64, integral_constant<int, 8>{}, m);
          else if (one_wave && vecs <= 1024) launch(g64, integral_constant<int, 16>{}, m);
          else if (one_wave) launch(g64, integral_constant<int, 0>{}, m);
          // the loss alone of long rows: nothing to keep, and more rows under way (8192 rows of 131072 fp16 logits: 399 us, held 511)
          else if (h.k <= 256 && grad == nullptr && h.rows >= kComputeUnits) launch(g256, integral_constant<int, 0>{}, m);
          else if (h.k <= 256 && vecs <= 1024) launch(g256, integral_constant<int, 4>{}, m);
          else if (h.k <= 128 && vecs <= 2048 && many) launch(g128, integral_constant<int, 16>{}, m);  // 4134 rows of 8970 fp16 logits: 45 us, with g256 52
          else if (h.k <= 256 && vecs <= 2048) launch(g256, integral_constant<int, 8>{}, m);
          else if (h.k <= 256 && vecs <= 4096) launch(g256, integral_constant<int, 16>{}, m);
          else if (h.k <= 512 && vecs <= 8192) launch(g512, integral_constant<int, 16>{}, m);
          else if (vecs <= 16384) launch(g1024, integral_constant<int, 16>{}, m);
          else launch(g1024, integral_constant<int, 0>{}, m);
        };
        with_mix(mix_of(h.weight, h.temperature), pick);
      });
      check_launch("distill launch");
    }
    if (loss != nullptr && h.reduction != TDM_DISTILL_NONE) {
      hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(kFoldThreads), 0, st, a, loss);
      check_launch("distill_sum launch");
    }
  });
}

}  // extern "C"
