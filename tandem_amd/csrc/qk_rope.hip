// K6: the norm of every query and key head with the position rotation in the same pass, and its gradient.
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = r x w,  (a, b) -> (a c - b s, b c + a s)  with c, s = cos, sin(position * f_i)
//
// over a head's elements; (a, b) are elements i and i + R/2 of the R rotated ones, or 2i and 2i + 1 (interleaved), and the
// elements behind the rotated ones are normed only. With g the upstream gradient rotated back and u = r x,
//
//   dx = r (w g - u mean(w g u)),   dw = sum over tokens and heads of g u.
//
// The pass is bound by memory: x is read once and y (dx) written once, nothing is kept between the passes (r is recomputed from
// the x that the gradient reads anyway). A group of lanes takes a head: every lane holds whole pairs, so the rotation needs no
// exchange, and the sums need log2(lanes) steps. A workgroup takes a few tokens with all their heads, so that a token's
// angles are computed once, not once per head: in doubles up to the quarter turn (a float's angle would be off by whole
// radians at far positions), then in floats on a quarter turn.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/tandem_hip.h"
#include "common.h"
#include "ops_device.h"

namespace tandem_hip {
namespace ops {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMostTokens = 16;   // per workgroup and round
constexpr int kMostPairs = 256;   // heads of up to 512 elements
constexpr int kLdsPairs = 2048;   // tokens * pairs of one round
constexpr int kMostGroups = 1024; // workgroups of the gradient: one row of partial sums each

struct Heads {
  char* data;
  int64_t batch, token, head;  // strides, in elements
};

struct RopeArgs {
  Heads x[2], y[2];        // q, k: in; out (the gradient's: upstream)
  Heads dx[2];             // the gradient's result
  Heads dv, dv_out;        // copied from dv to dv_out, where there is one
  int heads[2];
  const void* weight[2];   // null: ones
  const void* positions;
  const double* inv_freq;
  float* partial;          // [workgroups][2][head_dim]
  int64_t batch_stride, token_stride;  // of positions
  uint32_t tokens, per_batch;          // in all; of a sequence
  int head_dim, rotary;
  int log_lanes;           // per head
  int round;               // tokens per workgroup and round
  int interleaved, weight_f32, position_i64;
  float eps;
};

// cos and sin of position * f: the quarter turns in doubles, the rest, at most an eighth of a turn, in floats.
__device__ __forceinline__ void turn(double position, double f, float& c, float& s) {
  const double quarters = position * (f * 0.63661977236758134308);  // 2 / pi
  const double whole = rint(quarters);
  float sn, cs;
  sincospif(0.5f * static_cast<float>(quarters - whole), &sn, &cs);
  const int q = static_cast<int>(static_cast<long long>(whole) & 3);
  c = q == 0 ? cs : q == 1 ? -sn : q == 2 ? -cs : sn;
  s = q == 0 ? sn : q == 1 ? cs : q == 2 ? -sn : -cs;
}

struct Shared {
  float cos[kLdsPairs], sin[kLdsPairs];
  float weight[2][2 * kMostPairs];
  uint32_t batch[kMostTokens], at[kMostTokens];
};

template <typename T>
__device__ __forceinline__ T* row_of(const Heads& h, const Shared& sh, int token, int head) {
  return reinterpret_cast<T*>(h.data) + sh.batch[token] * h.batch + sh.at[token] * h.token + head * h.head;
}

// A round's angles and places. `first`: its first token.
__device__ __forceinline__ void stage(const RopeArgs& a, Shared& sh, uint32_t first, int here) {
  const int pairs = a.head_dim / 2, turned = a.rotary / 2;
  if (threadIdx.x < static_cast<unsigned>(here)) {
    const uint32_t n = first + threadIdx.x;
    sh.batch[threadIdx.x] = n / a.per_batch;
    sh.at[threadIdx.x] = n % a.per_batch;
  }
  for (int i = threadIdx.x; i < here * pairs; i += kThreads) {
    const int t = i / pairs, p = i - t * pairs;
    float c = 1.0f, s = 0.0f;
    if (p < turned) {
      const uint32_t n = first + t;
      const int64_t at = (n / a.per_batch) * a.batch_stride + (n % a.per_batch) * a.token_stride;
      const double position = a.position_i64 ? static_cast<double>(static_cast<const int64_t*>(a.positions)[at])
                                             : static_cast<double>(static_cast<const int32_t*>(a.positions)[at]);
      turn(position, a.inv_freq[p], c, s);
    }
    sh.cos[i] = c;
    sh.sin[i] = s;
  }
}

template <typename T>
__device__ __forceinline__ void stage_weights(const RopeArgs& a, Shared& sh) {
  for (int i = threadIdx.x; i < 2 * a.head_dim; i += kThreads) {
    const int w = i >= a.head_dim, d = i - w * a.head_dim;
    float x = 1.0f;
    if (a.weight[w] != nullptr) x = a.weight_f32 ? static_cast<const float*>(a.weight[w])[d] : widen(static_cast<const T*>(a.weight[w])[d]);
    sh.weight[w][d] = x;
  }
}

// The pairs that a lane of a head's group holds: kC runs of kV pairs.
template <typename T, int kV, int kC>
struct Lane {
  using P = Pack<T, kV>;
  int first[kC];   // pair
  int a[kC], b[kC];  // the elements that the run's two accesses begin at
  bool on[kC];

  __device__ __forceinline__ Lane(const RopeArgs& args) {
    const int lanes = 1 << args.log_lanes, lane = threadIdx.x & (lanes - 1);
    const int pairs = args.head_dim / 2, turned = args.rotary / 2;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const int p = (c * lanes + lane) * kV;
      on[c] = p < pairs;
      first[c] = on[c] ? p : 0;
      if (args.interleaved) {
        a[c] = 2 * first[c];
        b[c] = a[c] + kV;
      } else {
        const bool in = first[c] < turned;
        a[c] = in ? first[c] : args.rotary + first[c] - turned;
        b[c] = a[c] + (in ? turned : pairs - turned);
      }
    }
  }

  // A run's elements as pairs (lo[i], hi[i]).
  __device__ __forceinline__ void load(const T* row, bool interleaved, float (&lo)[kC][kV], float (&hi)[kC][kV]) const {
    P ra[kC], rb[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      ra[c] = P::load(row + a[c]);
      rb[c] = P::load(row + b[c]);
    }
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      float x[2 * kV];
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        x[i] = on[c] ? widen(ra[c].v[i]) : 0.0f;
        x[kV + i] = on[c] ? widen(rb[c].v[i]) : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        lo[c][i] = interleaved ? x[2 * i] : x[i];
        hi[c][i] = interleaved ? x[2 * i + 1] : x[kV + i];
      }
    }
  }

  __device__ __forceinline__ void store(T* row, bool interleaved, const float (&lo)[kC][kV], const float (&hi)[kC][kV]) const {
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      P pa, pb;
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const float x = interleaved ? ((i & 1) ? hi[c][i / 2] : lo[c][i / 2]) : lo[c][i];
        const float y = interleaved ? (((kV + i) & 1) ? hi[c][(kV + i) / 2] : lo[c][(kV + i) / 2]) : hi[c][i];
        pa.v[i] = narrow<T>(x);
        pb.v[i] = narrow<T>(y);
      }
      if (on[c]) {
        pa.store(row + a[c]);
        pb.store(row + b[c]);
      }
    }
  }

  // The element of a head that lo[c][i] / hi[c][i] is.
  __device__ __forceinline__ int element(int c, int i, bool high, bool interleaved) const {
    if (interleaved) return a[c] + 2 * i + (high ? 1 : 0);
    return (high ? b[c] : a[c]) + i;
  }
};

__device__ __forceinline__ float group_sum(float x, int lanes) {
  for (int d = 1; d < lanes; d *= 2) x += __shfl_xor(x, d);
  return x;
}

template <typename T, int kV, int kC>
__global__ __launch_bounds__(kThreads) void qk_rope_kernel(RopeArgs a) {
  __shared__ Shared sh;
  const int lanes = 1 << a.log_lanes, groups = kThreads >> a.log_lanes;
  const int group = threadIdx.x >> a.log_lanes;
  const int pairs = a.head_dim / 2;
  const bool il = a.interleaved;
  const Lane<T, kV, kC> lane(a);
  const float inv_dim = 1.0f / static_cast<float>(a.head_dim);
  const uint32_t first = blockIdx.x * static_cast<uint32_t>(a.round);
  const int here = static_cast<int>(std::min<uint32_t>(a.round, a.tokens - first));
  stage(a, sh, first, here);
  stage_weights<T>(a, sh);
  __syncthreads();
  for (int w = 0; w < 2; ++w) {
    const int heads = a.heads[w], items = here * heads;
    for (int base = 0; base < items; base += groups) {
      const int item = base + group;
      const bool live = item < items;
      const int t = live ? item / heads : 0, h = live ? item - t * heads : 0;
      float lo[kC][kV], hi[kC][kV];
      lane.load(row_of<T>(a.x[w], sh, t, h), il, lo, hi);
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int i = 0; i < kV; ++i) sum += lo[c][i] * lo[c][i] + hi[c][i] * hi[c][i];
      const float r = rsqrtf(group_sum(sum, lanes) * inv_dim + a.eps);
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          const float cs = sh.cos[t * pairs + lane.first[c] + i], sn = sh.sin[t * pairs + lane.first[c] + i];
          const float x = lo[c][i] * r * sh.weight[w][lane.element(c, i, false, il)];
          const float y = hi[c][i] * r * sh.weight[w][lane.element(c, i, true, il)];
          lo[c][i] = x * cs - y * sn;
          hi[c][i] = y * cs + x * sn;
        }
      if (live) lane.store(row_of<T>(a.y[w], sh, t, h), il, lo, hi);
    }
  }
}

template <typename T, int kV, int kC>
__global__ __launch_bounds__(kThreads) void qk_rope_grad_kernel(RopeArgs a) {
  __shared__ Shared sh;
  __shared__ float s_dw[kWaves][2 * kMostPairs];
  const int lanes = 1 << a.log_lanes, groups = kThreads >> a.log_lanes;
  const int group = threadIdx.x >> a.log_lanes;
  const int pairs = a.head_dim / 2;
  const bool il = a.interleaved;
  const Lane<T, kV, kC> lane(a);
  const float inv_dim = 1.0f / static_cast<float>(a.head_dim);
  float dlo[2][kC][kV] = {}, dhi[2][kC][kV] = {};
  stage_weights<T>(a, sh);
  for (uint32_t first = blockIdx.x * static_cast<uint32_t>(a.round); first < a.tokens; first += gridDim.x * static_cast<uint32_t>(a.round)) {
    const int here = static_cast<int>(std::min<uint32_t>(a.round, a.tokens - first));
    __syncthreads();
    stage(a, sh, first, here);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int heads = a.heads[w], items = here * heads;
      for (int base = 0; base < items; base += groups) {
        const int item = base + group;
        const bool live = item < items;
        const int t = live ? item / heads : 0, h = live ? item - t * heads : 0;
        float lo[kC][kV], hi[kC][kV], glo[kC][kV] = {}, ghi[kC][kV] = {};
        lane.load(row_of<T>(a.x[w], sh, t, h), il, lo, hi);
        if (a.y[w].data != nullptr) lane.load(row_of<T>(a.y[w], sh, t, h), il, glo, ghi);
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < kC; ++c)
#pragma unroll
          for (int i = 0; i < kV; ++i) sum += lo[c][i] * lo[c][i] + hi[c][i] * hi[c][i];
        const float r = rsqrtf(group_sum(sum, lanes) * inv_dim + a.eps);
        float dot = 0.0f;
#pragma unroll
        for (int c = 0; c < kC; ++c)
#pragma unroll
          for (int i = 0; i < kV; ++i) {
            const float cs = sh.cos[t * pairs + lane.first[c] + i], sn = sh.sin[t * pairs + lane.first[c] + i];
            const float x = glo[c][i] * cs + ghi[c][i] * sn, y = ghi[c][i] * cs - glo[c][i] * sn;
            lo[c][i] *= r;
            hi[c][i] *= r;
            if (live) {
              dlo[w][c][i] += x * lo[c][i];
              dhi[w][c][i] += y * hi[c][i];
            }
            glo[c][i] = x * sh.weight[w][lane.element(c, i, false, il)];
            ghi[c][i] = y * sh.weight[w][lane.element(c, i, true, il)];
            dot += glo[c][i] * lo[c][i] + ghi[c][i] * hi[c][i];
          }
        dot = group_sum(dot, lanes) * inv_dim;
#pragma unroll
        for (int c = 0; c < kC; ++c)
#pragma unroll
          for (int i = 0; i < kV; ++i) {
            glo[c][i] = r * (glo[c][i] - lo[c][i] * dot);
            ghi[c][i] = r * (ghi[c][i] - hi[c][i] * dot);
          }
        if (live) lane.store(row_of<T>(a.dx[w], sh, t, h), il, glo, ghi);
      }
    }
    if (a.dv_out.data != nullptr) {
      const int heads = a.heads[1], items = here * heads;
      for (int item = group; item < items; item += groups) {
        const int t = item / heads, h = item - t * heads;
        using P = Pack<T, kV>;
        T* to = row_of<T>(a.dv_out, sh, t, h);
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          if (!lane.on[c]) continue;
          P pa{}, pb{};
          if (a.dv.data != nullptr) {
            const T* from = row_of<T>(a.dv, sh, t, h);
            pa = P::load(from + lane.a[c]);
            pb = P::load(from + lane.b[c]);
          }
          pa.store(to + lane.a[c]);
          pb.store(to + lane.b[c]);
        }
      }
    }
  }
  // the workgroup's sums of the weights' gradients: over the groups of a wave, then over the waves, always in this order
  const int wave = threadIdx.x / kWave;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        float x = dlo[w][c][i], y = dhi[w][c][i];
        for (int d = lanes; d < kWave; d *= 2) {
          x += __shfl_xor(x, d);
          y += __shfl_xor(y, d);
        }
        if (lane.on[c] && (threadIdx.x % kWave) < static_cast<unsigned>(lanes)) {
          s_dw[wave][lane.element(c, i, false, il)] = x;
          s_dw[wave][lane.element(c, i, true, il)] = y;
        }
      }
    __syncthreads();
    for (int d = threadIdx.x; d < a.head_dim; d += kThreads) {
      float x = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) x += s_dw[k][d];
      a.partial[(static_cast<int64_t>(blockIdx.x) * 2 + w) * a.head_dim + d] = x;
    }
  }
}

// dw = the sum of the workgroups' rows, in order: 16 stretches of rows side by side, then the 16.
constexpr int kFoldLanes = 64, kFoldRows = 16;
template <typename T>
__global__ __launch_bounds__(kFoldLanes* kFoldRows) void qk_rope_fold_kernel(const float* partial, int rows, int head_dim, int f32, void* dq_weight,
                                                                             void* dk_weight) {
  __shared__ float s_sum[kFoldRows][kFoldLanes];
  const int lane = threadIdx.x % kFoldLanes, part = threadIdx.x / kFoldLanes;
  const int col = static_cast<int>(blockIdx.x) * kFoldLanes + lane;
  const int per = (rows + kFoldRows - 1) / kFoldRows;
  float x = 0.0f;
  if (col < 2 * head_dim)
    for (int r = part * per; r < std::min(rows, (part + 1) * per); ++r) x += partial[static_cast<int64_t>(r) * 2 * head_dim + col];
  s_sum[part][lane] = x;
  __syncthreads();
  if (part != 0 || col >= 2 * head_dim) return;
  x = 0.0f;
#pragma unroll
  for (int p = 0; p < kFoldRows; ++p) x += s_sum[p][lane];
  void* to = col < head_dim ? dq_weight : dk_weight;
  if (to == nullptr) return;
  const int d = col < head_dim ? col : col - head_dim;
  if (f32) static_cast<float*>(to)[d] = x;
  else static_cast<T*>(to)[d] = narrow<T>(x);
}

// ---------------------------------------------------------------- host

int64_t groups_of(const tdm_qk_shape& s, int round) {
  return std::min<int64_t>((s.batch * s.tokens + round - 1) / round, kMostGroups);
}

// Tokens per workgroup and round: enough for every group of lanes to have four heads, as long as there are workgroups for
// the whole GPU.
int round_of(const tdm_qk_shape& s, int groups) {
  const int64_t tokens = s.batch * s.tokens;
  int round = 1;
  while (round < kMostTokens && round * 2 * (s.head_dim / 2) <= kLdsPairs && round * (s.q_heads + s.kv_heads) < 4 * groups && tokens / (round * 2) >= 1024) round *= 2;
  return round;
}

void check_shape(const tdm_qk_shape* s) {
  require(s != nullptr, "qk_norm_rope: null shape");
  require(operator_dtype(s->dtype), "qk_norm_rope: the dtype must be float32, float16 or bfloat16");
  require(s->weight_dtype == s->dtype || s->weight_dtype == TDM_F32, "qk_norm_rope: weights of the heads' dtype or float32");
  require(s->position_dtype == TDM_I64 || s->position_dtype == TDM_I32, "qk_norm_rope: positions must be int64 or int32");
  require(s->batch >= 0 && s->tokens >= 0 && s->batch < (int64_t(1) << 31) && s->tokens < (int64_t(1) << 31) && s->batch * s->tokens < (int64_t(1) << 31),
          "qk_norm_rope: 0 to 2^31 - 1 tokens");
  require(s->q_heads >= 0 && s->kv_heads >= 0 && s->q_heads <= 65536 && s->kv_heads <= 65536, "qk_norm_rope: 0 to 65536 heads");
  require(s->head_dim >= 2 && s->head_dim <= 2 * kMostPairs && s->head_dim % 2 == 0, "qk_norm_rope: heads of 2 to 512 elements, an even number");
  require(s->rotary_dim >= 0 && s->rotary_dim <= s->head_dim && s->rotary_dim % 2 == 0, "qk_norm_rope: an even number of rotated elements, at most the head's");
  require(s->eps >= 0.0f, "qk_norm_rope: eps must not be negative");
}

struct Plan {
  RopeArgs args{};
  int run = 1;  // kV
  uintptr_t bits = 0;

  Heads heads(const tdm_heads* h, int es) {
    Heads r{static_cast<char*>(h->data), h->batch_stride, h->token_stride, h->head_stride};
    if (r.data != nullptr)
      bits |= reinterpret_cast<uintptr_t>(r.data) | static_cast<uintptr_t>((r.batch | r.token | r.head) * es);
    return r;
  }
};

void finish(Plan& p, const tdm_qk_shape& s, const tdm_positions* at, const double* inv_freq) {
  RopeArgs& a = p.args;
  require(s.rotary_dim == 0 || (at != nullptr && at->data != nullptr && inv_freq != nullptr), "qk_norm_rope: null pointer");
  if (at != nullptr) {
    a.positions = at->data;
    a.batch_stride = at->batch_stride;
    a.token_stride = at->token_stride;
  }
  a.inv_freq = inv_freq;
  a.heads[0] = s.q_heads;
  a.heads[1] = s.kv_heads;
  a.tokens = static_cast<uint32_t>(s.batch * s.tokens);
  a.per_batch = static_cast<uint32_t>(std::max<int64_t>(s.tokens, 1));
  a.head_dim = s.head_dim;
  a.rotary = s.rotary_dim;
  a.interleaved = s.interleaved != 0;
  a.weight_f32 = s.weight_dtype == TDM_F32;
  a.position_i64 = s.position_dtype == TDM_I64;
  a.eps = s.eps;
  // the longest run of pairs, 16 bytes at most, that every address allows and that does not straddle the end of the rotated pairs
  const int es = s.dtype == TDM_F32 ? 4 : 2, pairs = s.head_dim / 2, turned = s.rotary_dim / 2;
  int run = access_width(p.bits, es) / es;
  const int whole = a.interleaved ? pairs : (turned | (pairs - turned));
  while (run > 1 && whole % run != 0) run /= 2;
  p.run = run;
  const int runs = run == 1 ? 4 : run == 2 ? 2 : 1;  // kC
  while ((1 << a.log_lanes) * run * runs < pairs) ++a.log_lanes;
  a.round = round_of(s, kThreads >> a.log_lanes);
}

template <class F>
void with_run(int run, F&& f) {
  switch (run) {
    case 8: f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{}); return;
    case 4: f(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{}); return;
    case 2: f(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{}); return;
    default: f(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{}); return;
  }
}

}  // namespace

}  // namespace ops
}  // namespace tandem_hip

using namespace tandem_hip;
using namespace tandem_hip::ops;

extern "C" {

int tdm_k6_qk_norm_rope(const tdm_qk_shape* shape, const tdm_heads* q, const tdm_heads* k, const void* q_weight, const void* k_weight,
                        const tdm_positions* positions, const double* inv_freq, const tdm_heads* q_out, const tdm_heads* k_out,
                        tdm_stream stream) {
  return guard([&] {
    check_shape(shape);
    const tdm_qk_shape& s = *shape;
    if (s.batch * s.tokens == 0 || s.q_heads + s.kv_heads == 0) return;
    require(q != nullptr && k != nullptr && q_out != nullptr && k_out != nullptr, "qk_norm_rope: null pointer");
    require((s.q_heads == 0 || (q->data != nullptr && q_out->data != nullptr)) && (s.kv_heads == 0 || (k->data != nullptr && k_out->data != nullptr)),
            "qk_norm_rope: null pointer");
    const int es = s.dtype == TDM_F32 ? 4 : 2;
    Plan p;
    p.args.x[0] = p.heads(q, es);
    p.args.x[1] = p.heads(k, es);
    p.args.y[0] = p.heads(q_out, es);
    p.args.y[1] = p.heads(k_out, es);
    p.args.weight[0] = q_weight;
    p.args.weight[1] = k_weight;
    finish(p, s, positions, inv_freq);
    const dim3 grid((p.args.tokens + p.args.round - 1) / p.args.round);
    require(grid.x < (1u << 24), "qk_norm_rope: 2^24 workgroups or more");
    with_dtype(s.dtype, [&](auto t) {
      using T = decltype(t);
      with_run(p.run, [&](auto v, auto c) {
        if constexpr (v.value * sizeof(T) <= 16)
          hipLaunchKernelGGL((qk_rope_kernel<T, v.value, c.value>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), p.args);
      });
    });
    check_launch("qk_rope launch");
  });
}

int64_t tdm_k6_qk_norm_rope_grad_workspace(const tdm_qk_shape* shape) {
  int64_t bytes = -1;
  guard([&] {
    check_shape(shape);
    bytes = groups_of(*shape, 1) * 2 * shape->head_dim * 4;
  });
  return bytes;
}

int tdm_k6_qk_norm_rope_grad(const tdm_qk_shape* shape, const tdm_heads* dq_out, const tdm_heads* dk_out, const tdm_heads* dv_out,
                             const tdm_heads* q, const tdm_heads* k, const void* q_weight, const void* k_weight,
                             const tdm_positions* positions, const double* inv_freq, const tdm_heads* dq, const tdm_heads* dk,
                             const tdm_heads* dv, void* dq_weight, void* dk_weight, void* workspace, int64_t workspace_bytes,
                             tdm_stream stream) {
  return guard([&] {
    check_shape(shape);
    const tdm_qk_shape& s = *shape;
    const bool nothing = s.batch * s.tokens == 0 || s.q_heads + s.kv_heads == 0;
    require(dq_out != nullptr && dk_out != nullptr && q != nullptr && k != nullptr && dq != nullptr && dk != nullptr, "qk_norm_rope_grad: null pointer");
    require(nothing || s.q_heads == 0 || (q->data != nullptr && dq->data != nullptr), "qk_norm_rope_grad: null pointer");
    require(nothing || s.kv_heads == 0 || (k->data != nullptr && dk->data != nullptr), "qk_norm_rope_grad: null pointer");
    const int es = s.dtype == TDM_F32 ? 4 : 2;
    Plan p;
    p.args.x[0] = p.heads(q, es);
    p.args.x[1] = p.heads(k, es);
    p.args.y[0] = p.heads(dq_out, es);
    p.args.y[1] = p.heads(dk_out, es);
    p.args.dx[0] = p.heads(dq, es);
    p.args.dx[1] = p.heads(dk, es);
    if (dv != nullptr && dv->data != nullptr) {
      p.args.dv_out = p.heads(dv, es);
      if (dv_out != nullptr) p.args.dv = p.heads(dv_out, es);
    }
    p.args.weight[0] = q_weight;
    p.args.weight[1] = k_weight;
    p.args.weight_f32 = s.weight_dtype == TDM_F32;
    if (!nothing) finish(p, s, positions, inv_freq);
    const int64_t groups = nothing ? 0 : groups_of(s, p.args.round);
    require(groups == 0 || (workspace != nullptr && workspace_bytes >= groups * 2 * s.head_dim * 4 && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
            "qk_norm_rope_grad: the workspace starts on 16 bytes and holds tdm_k6_qk_norm_rope_grad_workspace bytes");
    p.args.partial = static_cast<float*>(workspace);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    with_dtype(s.dtype, [&](auto t) {
      using T = decltype(t);
      if (groups > 0) {
        with_run(p.run, [&](auto v, auto c) {
          if constexpr (v.value * sizeof(T) <= 16)
            hipLaunchKernelGGL((qk_rope_grad_kernel<T, v.value, c.value>), dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, st, p.args);
        });
        check_launch("qk_rope_grad launch");
      }
      if (dq_weight != nullptr || dk_weight != nullptr) {
        hipLaunchKernelGGL((qk_rope_fold_kernel<T>), dim3((2 * s.head_dim + kFoldLanes - 1) / kFoldLanes), dim3(kFoldLanes * kFoldRows), 0, st,
                           static_cast<const float*>(workspace), static_cast<int>(groups), s.head_dim, p.args.weight_f32, dq_weight, dk_weight);
        check_launch("qk_rope_fold launch");
      }
    });
  });
}

}  // extern "C"
