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
  const float* count;      // rows that count, the mean's divisor; null: `divisor`
  int64_t rows, vocab, ignore;
  int k, index_i64, teacher_dtype, targets_i64;
  int upstream_step;       // 0: one value for all rows
  int keep_ones;           // where the upstream value is 1, the gradient there already is right
  float temperature, weight, scale, divisor;
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float ln_of(float x) { return __builtin_amdgcn_logf(x) * kLn2; }

// Sum or maximum over the kG lanes of a row; every lane gets it. `s`: kG / 64 floats of LDS that nothing else uses.
template <int kG, class F>
__device__ __forceinline__ float over_row(float x, float* s, F f) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) x = f(x, __shfl_xor(x, d));
  if constexpr (kG > kWave) {
    __syncthreads();
    if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = x;
    __syncthreads();
    x = s[0];
#pragma unroll
    for (int w = 1; w < kG / kWave; ++w) x = f(x, s[w]);
  }
  return x;
}
struct Add { __device__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };

__device__ __forceinline__ float teacher_logit(const DistillArgs& a, int64_t at) {
  if (a.teacher_dtype == TDM_F32) return static_cast<const float*>(a.teacher)[at];
  if (a.teacher_dtype == TDM_F16) return static_cast<float>(static_cast<const _Float16*>(a.teacher)[at]);
  return static_cast<float>(static_cast<const __bf16*>(a.teacher)[at]);
}

__device__ __forceinline__ int64_t index_of(const void* p, int i64, int64_t at) {
  return i64 ? static_cast<const int64_t*>(p)[at] : static_cast<int64_t>(static_cast<const int32_t*>(p)[at]);
}

// A workgroup of kG lanes per row. kMix: both temperatures are needed (a < 1 and T != 1).
// LDS: kG / 64 floats, then k + 1 columns and k + 1 values.
template <typename T, int kG, bool kMix>
__global__ __launch_bounds__(kG) void distill_kernel(DistillArgs a) {
  constexpr int kN = 16 / static_cast<int>(sizeof(T));
  using P = Pack<T, kN>;
  extern __shared__ float lds[];
  float* const s_red = lds;
  int32_t* const s_col = reinterpret_cast<int32_t*>(lds + 16);
  float* const s_val = lds + 16 + a.k + 1;
  const int tid = threadIdx.x;
  const float lowest = -__builtin_inff();
  const float inv_t = 1.0f / a.temperature, c_t = kLog2e * inv_t;
  // without kMix one exponential does for both parts: at T where a = 1, at 1 where a = 0 or T = 1 (c_t is then log2(e) too)
  const float c = kMix || a.weight > 0.0f ? c_t : kLog2e;

  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float up = a.upstream == nullptr ? 1.0f : a.upstream[row * a.upstream_step];
    if (a.keep_ones && up == 1.0f) continue;
    const T* const x = static_cast<const T*>(a.logits) + row * a.vocab;
    T* const g = a.grad == nullptr ? nullptr : static_cast<T*>(a.grad) + row * a.vocab;
    const int64_t y = a.targets == nullptr ? 0 : index_of(a.targets, a.targets_i64, row);
    const bool counted = a.targets == nullptr || y != a.ignore;
    // the row's elements before its first whole vector, and its vectors
    const int head = static_cast<int>(std::min<int64_t>(a.vocab, ((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    const int64_t vecs = (a.vocab - head) / kN;
    const int tail = static_cast<int>(a.vocab - head - vecs * kN);
    const int64_t edge = tid < head ? tid : tid - head < tail ? head + vecs * kN + (tid - head) : -1;  // this lane's single element
    if (!counted) {
      if (a.rows_loss != nullptr && tid == 0) a.rows_loss[row] = 0.0f;
      if (g != nullptr) {
        P zero;
#pragma unroll
        for (int i = 0; i < kN; ++i) zero.v[i] = narrow<T>(0.0f);
        for (int64_t v = tid; v < vecs; v += kG) zero.store(g + head + v * kN);
        if (edge >= 0) g[edge] = narrow<T>(0.0f);
      }
      continue;
    }

    // the teacher
    const bool soft = a.weight > 0.0f, hard = a.weight < 1.0f;
    float bad = hard && (y < 0 || y >= a.vocab) ? 1.0f : 0.0f;
    float t_max = lowest;
    __syncthreads();  // the last row's columns and values have been read
    if (soft)
      for (int i = tid; i < a.k; i += kG) {
        const int64_t j = index_of(a.index, a.index_i64, row * a.k + i);
        float t = teacher_logit(a, row * a.k + i);
        if (j < 0) t = lowest;
        if (j >= a.vocab || t != t) bad = 1.0f;
        s_col[i] = j < 0 || j >= a.vocab ? -1 : static_cast<int32_t>(j);
        s_val[i] = t;
        t_max = fmaxf(t_max, t);
      }
    t_max = over_row<kG>(t_max, s_red, Max{});
    bad = over_row<kG>(bad, s_red, Max{});
    const bool taught = soft && t_max != lowest;  // else no entry says anything
    float t_sum = 0.0f;
    if (taught)
      for (int i = tid; i < a.k; i += kG) {
        s_val[i] = (s_val[i] - t_max) * inv_t;
        t_sum += exp2_of(s_val[i] * kLog2e);
      }
    t_sum = over_row<kG>(t_sum, s_red, Add{});

    // the student's maximum and sums, running: z at exponents c (x - m), z1 at log2(e) (x - m)
    float m = lowest, z = 0.0f, z1 = 0.0f;
    auto take = [&](float xm, auto each, int n) {  // n elements whose maximum is xm
      const float top = fmaxf(m, xm);
      const float base = top == lowest ? 0.0f : top;
      z *= exp2_of((m - base) * c);
      if (kMix) z1 *= exp2_of((m - base) * kLog2e);
      m = top;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        z += exp2_of((each(i) - base) * c);
        if (kMix) z1 += exp2_of((each(i) - base) * kLog2e);
      }
    };
    for (int64_t v = tid; v < vecs; v += kG) {
      const P p = P::load(x + head + v * kN);
      float f[kN], xm = lowest;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        f[i] = widen(p.v[i]);
        xm = fmaxf(xm, f[i]);
      }
      take(xm, [&](int i) { return f[i]; }, kN);
    }
    if (edge >= 0) {
      const float f = widen(x[edge]);
      take(f, [&](int) { return f; }, 1);
    }
    const float top = over_row<kG>(m, s_red, Max{});
    const float base = top == lowest ? 0.0f : top;
    z *= exp2_of((m - base) * c);
    z = over_row<kG>(z, s_red, Add{});
    if (kMix) {
      z1 *= exp2_of((m - base) * kLog2e);
      z1 = over_row<kG>(z1, s_red, Add{});
    } else {
      z1 = z;
    }
    const float wrong = bad != 0.0f ? __builtin_nanf("") : 0.0f;  // a column outside the vocabulary shows

    // the loss
    const float t2 = a.temperature * a.temperature;
    float part = 0.0f;
    const float log_z = ln_of(z), log_t = ln_of(t_sum), p_scale = 1.0f / t_sum;
    if (taught)
      for (int i = tid; i < a.k; i += kG) {
        const float t = s_val[i], p = exp2_of(t * kLog2e) * p_scale;
        const int j = s_col[i];
        if (!(p == 0.0f) && j >= 0) part += p * (t - log_t - (widen(x[j]) - top) * inv_t + log_z);
        s_val[i] = j >= 0 ? p : 0.0f;
      }
    part *= a.weight * t2;
    if (hard && tid == 0 && bad == 0.0f) part += (1.0f - a.weight) * (ln_of(z1) - (widen(x[y]) - top));
    if (a.rows_loss != nullptr) {
      part = over_row<kG>(part, s_red, Add{});
      if (tid == 0) a.rows_loss[row] = part + wrong;
    }
    if (g == nullptr) continue;

    // the gradient: every element from the sums, then the teacher's columns and the target again, with what they take off
    const float s = a.scale * up / (a.count == nullptr ? a.divisor : *a.count) + wrong;
    const float w_t = taught ? s * a.weight * a.temperature : 0.0f, w_1 = hard ? s * (1.0f - a.weight) : 0.0f;
    const float k_t = (kMix ? w_t : w_t + w_1) / z, k_1 = w_1 / z1;
    auto slope = [&](float f) {
      float e = k_t * exp2_of((f - top) * c);
      if (kMix) e += k_1 * exp2_of((f - top) * kLog2e);
      return e;
    };
    for (int64_t v = tid; v < vecs; v += kG) {
      P p = P::load(x + head + v * kN);
#pragma unroll
      for (int i = 0; i < kN; ++i) p.v[i] = narrow<T>(slope(widen(p.v[i])));
      p.store(g + head + v * kN);
    }
    if (edge >= 0) g[edge] = narrow<T>(slope(widen(x[edge])));
    if (tid == 0) {
      s_col[a.k] = hard && bad == 0.0f ? static_cast<int32_t>(y) : -1;
      s_val[a.k] = hard ? w_1 : 0.0f;
    }
    __syncthreads();
    if (bad == 0.0f)
      for (int i = tid; i <= a.k; i += kG) {
        const int j = i == a.k ? s_col[a.k] : taught ? s_col[i] : -1;
        if (j < 0) continue;
        float off = 0.0f;  // all that falls on this column: an entry named twice, or the target's, comes out the same for each
        if (taught)
          for (int e = 0; e < a.k; ++e) off += s_col[e] == j ? w_t * s_val[e] : 0.0f;
        if (s_col[a.k] == j) off += s_val[a.k];
        g[j] = narrow<T>(slope(widen(x[j])) - off);
      }
  }
}

constexpr int kFoldThreads = 1024;

__device__ __forceinline__ float block_sum(float x, float* s) {
  return over_row<kFoldThreads>(x, s, Add{});
}

// How many rows count (at least one: a batch without any has loss 0).
__global__ __launch_bounds__(kFoldThreads) void distill_count_kernel(const void* targets, int i64, int64_t rows, int64_t ignore, float* count) {
  __shared__ float s[kFoldThreads / kWave];
  float n = 0.0f;
  for (int64_t r = threadIdx.x; r < rows; r += kFoldThreads) n += index_of(targets, i64, r) != ignore ? 1.0f : 0.0f;
  n = block_sum(n, s);
  if (threadIdx.x == 0) *count = fmaxf(n, 1.0f);
}

__global__ __launch_bounds__(kFoldThreads) void distill_sum_kernel(const float* rows_loss, int64_t rows, const float* count, float divisor, float* loss) {
  __shared__ float s[kFoldThreads / kWave];
  float x = 0.0f;
  for (int64_t r = threadIdx.x; r < rows; r += kFoldThreads) x += rows_loss[r];
  x = block_sum(x, s);
  if (threadIdx.x == 0) *loss = x / (count == nullptr ? divisor : *count);
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

constexpr int64_t kCountBytes = 256;

int64_t workspace_bytes_of(const tdm_distill_how& h) { return kCountBytes + (h.reduction == TDM_DISTILL_NONE ? 0 : h.rows * 4); }

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
    require(h.weight == 1.0f || targets != nullptr, "distill: a weight below 1 needs targets");
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
    if (mean && targets != nullptr) {
      hipLaunchKernelGGL(distill_count_kernel, dim3(1), dim3(kFoldThreads), 0, st, targets, h.target_dtype == TDM_I64, h.rows, h.ignore_index, count);
      check_launch("distill_count launch");
    }
    DistillArgs a{};
    a.logits = logits;
    a.index = teacher_index;
    a.teacher = teacher_logits;
    a.targets = targets;
    a.rows_loss = loss == nullptr ? nullptr : h.reduction == TDM_DISTILL_NONE ? loss : rows_loss;
    a.grad = grad;
    a.upstream = upstream;
    a.count = mean && targets != nullptr ? count : nullptr;
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
    if (h.rows > 0) {
      const bool mix = h.weight > 0.0f && h.weight < 1.0f && h.temperature != 1.0f;
      const unsigned lds = (16 + 2 * (h.k + 1)) * 4;
      with_dtype(h.dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t vecs = h.vocab * static_cast<int64_t>(sizeof(T)) / 16;
        auto launch = [&](auto g, auto m) {
          hipLaunchKernelGGL((distill_kernel<T, g.value, m.value>), dim3(static_cast<unsigned>(std::min<int64_t>(h.rows, 1 << 20))), dim3(g.value), lds, st, a);
        };
        auto pick = [&](auto m) {
          if (vecs <= 128) launch(std::integral_constant<int, 64>{}, m);
          else if (vecs <= 2048) launch(std::integral_constant<int, 256>{}, m);
          else launch(std::integral_constant<int, 1024>{}, m);
        };
        if (mix) pick(std::true_type{});
        else pick(std::false_type{});
      });
      check_launch("distill launch");
    }
    if (loss != nullptr && h.reduction != TDM_DISTILL_NONE) {
      hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(kFoldThreads), 0, st, rows_loss, h.rows, a.count, a.divisor, loss);
      check_launch("distill_sum launch");
    }
  });
}

}  // extern "C"
