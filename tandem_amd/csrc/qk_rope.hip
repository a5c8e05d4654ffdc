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
// radians at far positions), then in floats on a quarter turn. Queries and keys are different workgroups' work: one loop over one kind's
// heads, with one set of weights and sums in registers (both kinds in one workgroup cost the gradient 218 registers, two waves per SIMD).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "../../include/tandem_hip.h"
#include "common.h"
#include "ops_device.h"

namespace tandem_hip {
namespace ops {

namespace {

constexpr int kThreads = 256;
constexpr int kMostTokens = 32;   // per workgroup and round
constexpr int kMostPairs = 256;   // heads of up to 512 elements
constexpr int kLdsPairs = 2048;   // tokens * pairs of one round
constexpr int kGradGroups = 1536;  // workgroups of the gradient: twice what the GPU holds at once (three waves per SIMD)
constexpr int kMostGroups = 1024; // of one kind, at most: one row of partial sums each

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
  float* partial;          // [workgroups][head_dim]
  int64_t batch_stride, token_stride;  // of positions
  uint32_t tokens, per_batch;          // in all; of a sequence
  int head_dim, rotary;
  int log_lanes;           // per head
  int log_share[2];        // groups of lanes that share a token
  int round[2];            // tokens per workgroup and round
  uint32_t groups[2];      // workgroups of each kind: those of q first
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
  float weight[2 * kMostPairs];
};

// A token's heads.
template <typename T>
__device__ __forceinline__ T* row_of(const Heads& h, uint32_t batch, uint32_t at) {
  return reinterpret_cast<T*>(h.data) + batch * h.batch + at * h.token;
}

// A round's angles. `first`: its first token.
__device__ __forceinline__ void stage(const RopeArgs& a, Shared& sh, uint32_t first, int here) {
  const int pairs = a.head_dim / 2, turned = a.rotary / 2;
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
__device__ __forceinline__ void stage_weights(const RopeArgs& a, Shared& sh, int w) {
  const void* const weight = a.weight[w];
  for (int d = threadIdx.x; d < a.head_dim; d += kThreads)
    sh.weight[d] = weight == nullptr ? 1.0f : a.weight_f32 ? static_cast<const float*>(weight)[d] : widen(static_cast<const T*>(weight)[d]);
}

// The pairs that a lane of a head's group holds: kC runs of kV pairs.
template <typename T, int kV, int kC, bool kInterleaved>
struct Lane {
  using P = Pack<T, kV>;
  struct Raw {
    P a[kC], b[kC];
  };
  int first[kC];     // pair
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
      if (kInterleaved) {
        a[c] = 2 * first[c];
        b[c] = a[c] + kV;
      } else {
        const bool in = first[c] < turned;
        a[c] = in ? first[c] : args.rotary + first[c] - turned;
        b[c] = a[c] + (in ? turned : pairs - turned);
      }
    }
  }

  __device__ __forceinline__ Raw load(const T* row, bool there) const {  // zeros where there is nothing
    Raw r{};
#pragma unroll
    for (int c = 0; c < kC; ++c)
      if (there && on[c]) {
        r.a[c] = P::load(row + a[c]);
        r.b[c] = P::load(row + b[c]);
      }
    return r;
  }

  // A run's elements as pairs (lo[i], hi[i]).
  __device__ __forceinline__ void pairs_of(const Raw& r, float (&lo)[kC][kV], float (&hi)[kC][kV]) const {
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      float x[2 * kV];
      r.a[c].get(x);
      r.b[c].get(x + kV);
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        lo[c][i] = kInterleaved ? x[2 * i] : x[i];
        hi[c][i] = kInterleaved ? x[2 * i + 1] : x[kV + i];
      }
    }
  }

  __device__ __forceinline__ void store(T* row, const float (&lo)[kC][kV], const float (&hi)[kC][kV]) const {
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      P pa, pb;
      float x[2 * kV];
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        x[i] = kInterleaved ? ((i & 1) ? hi[c][i / 2] : lo[c][i / 2]) : lo[c][i];
        x[kV + i] = kInterleaved ? (((kV + i) & 1) ? hi[c][(kV + i) / 2] : lo[c][(kV + i) / 2]) : hi[c][i];
      }
      pa.set(x);
      pb.set(x + kV);
      if (on[c]) {
        pa.store_nt(row + a[c]);
        pb.store_nt(row + b[c]);
      }
    }
  }

  // The element of a head that lo[c][i] / hi[c][i] is.
  __device__ __forceinline__ int element(int c, int i, bool high) const {
    if (kInterleaved) return a[c] + 2 * i + (high ? 1 : 0);
    return (high ? b[c] : a[c]) + i;
  }

  // What every head of a token shares, and every head of its kind.
  __device__ __forceinline__ void angles(const Shared& sh, int at, float (&cs)[kC][kV], float (&sn)[kC][kV]) const {
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        cs[c][i] = sh.cos[at + first[c] + i];
        sn[c][i] = sh.sin[at + first[c] + i];
      }
  }
  __device__ __forceinline__ void weights(const float* w, float (&lo)[kC][kV], float (&hi)[kC][kV]) const {
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        lo[c][i] = w[element(c, i, false)];
        hi[c][i] = w[element(c, i, true)];
      }
  }
};

template <int kCtrl>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kCtrl, 0xf, 0xf, true));
}
// Over a head's lanes, every lane gets it: neighbours, pairs, mirrored quads and eights, then across rows of 16.
__device__ __forceinline__ float group_sum(float x, int log_lanes) {
  if (log_lanes >= 1) x = dpp_add<0xb1>(x);
  if (log_lanes >= 2) x = dpp_add<0x4e>(x);
  if (log_lanes >= 3) x = dpp_add<0x141>(x);
  if (log_lanes >= 4) x = dpp_add<0x140>(x);
  if (log_lanes >= 5) x += __shfl_xor(x, 16);
  if (log_lanes >= 6) x += __shfl_xor(x, 32);
  return x;
}

// What a workgroup works on: q or k (w), and which of that kind's workgroups it is.
struct Part {
  int w, heads, share, round;
  uint32_t index, of;
};
__device__ __forceinline__ Part part_of(const RopeArgs& a) {
  const int w = blockIdx.x >= a.groups[0];
  return Part{w, a.heads[w], 1 << a.log_share[w], a.round[w], blockIdx.x - (w ? a.groups[0] : 0u), a.groups[w]};
}

// A round: `round` tokens, each of them shared by `share` groups of lanes that take its heads in turn. The next head's elements
// are on their way while one is computed.
// 32768 tokens of 32 + 8 bf16 heads of 128 take 127 us, 5.3 TB/s of heads read and written; 16 such tokens 4.5 us, one round's latency.
template <typename T, int kV, int kC, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void qk_rope_kernel(RopeArgs a) {
  __shared__ Shared sh;
  using L = Lane<T, kV, kC, kInterleaved>;
  const Part part = part_of(a);
  const int group = threadIdx.x >> a.log_lanes;
  const L lane(a);
  const float inv_dim = 1.0f / static_cast<float>(a.head_dim);
  const uint32_t first = part.index * static_cast<uint32_t>(part.round);
  const int here = static_cast<int>(std::min<uint32_t>(part.round, a.tokens - first));
  const int t = group >> a.log_share[part.w];
  int left = t < here ? part.heads - (group & (part.share - 1)) : 0;  // of this group's heads: every part.share-th one
  const uint32_t token = first + std::min(t, here - 1), batch = token / a.per_batch, at = token % a.per_batch;
  const int64_t h0 = group & (part.share - 1);
  const Heads in = a.x[part.w], out = a.y[part.w];
  const T* x = row_of<T>(in, batch, at) + h0 * in.head;
  T* y = row_of<T>(out, batch, at) + h0 * out.head;
  const int64_t x_step = part.share * in.head, y_step = part.share * out.head;
  typename L::Raw next = lane.load(x, left > 0);
  stage(a, sh, first, here);
  stage_weights<T>(a, sh, part.w);
  __syncthreads();
  float cs[kC][kV], sn[kC][kV], wlo[kC][kV], whi[kC][kV];
  lane.angles(sh, std::min(t, here - 1) * (a.head_dim / 2), cs, sn);
  lane.weights(sh.weight, wlo, whi);
  for (int base = 0; base < part.heads; base += part.share, left -= part.share, x += x_step, y += y_step) {
    const typename L::Raw raw = next;
    next = lane.load(x + x_step, left > part.share);
    float lo[kC][kV], hi[kC][kV];
    lane.pairs_of(raw, lo, hi);
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int i = 0; i < kV; ++i) sum = fmaf(lo[c][i], lo[c][i], fmaf(hi[c][i], hi[c][i], sum));
    const float r = rsqrtf(fmaf(group_sum(sum, a.log_lanes), inv_dim, a.eps));
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const float p = lo[c][i] * r * wlo[c][i], q = hi[c][i] * r * whi[c][i];
        lo[c][i] = fmaf(p, cs[c][i], -(q * sn[c][i]));
        hi[c][i] = fmaf(q, cs[c][i], p * sn[c][i]);
      }
    if (left > 0) lane.store(y, lo, hi);
  }
}

// The same tokens' gradient takes 235 us: 1.14 GB with the values' copy, 4.9 TB/s, at three waves per SIMD. A workgroup stays for many rounds, so that the
// weights' sums leave its registers once.
template <typename T, int kV, int kC, bool kInterleaved>
__global__ __launch_bounds__(kThreads, 3) void qk_rope_grad_kernel(RopeArgs a) {
  __shared__ Shared sh;
  __shared__ float s_dw[2 * kMostPairs];
  using L = Lane<T, kV, kC, kInterleaved>;
  const Part part = part_of(a);
  const int group = threadIdx.x >> a.log_lanes;
  const L lane(a);
  const float inv_dim = 1.0f / static_cast<float>(a.head_dim);
  const int64_t h0 = group & (part.share - 1);
  const Heads in = a.x[part.w], up = a.y[part.w], out = a.dx[part.w];
  const bool given = up.data != nullptr;
  const int64_t x_step = part.share * in.head, g_step = part.share * up.head, o_step = part.share * out.head;
  float wlo[kC][kV], whi[kC][kV], dlo[kC][kV] = {}, dhi[kC][kV] = {};
  stage_weights<T>(a, sh, part.w);
  __syncthreads();
  lane.weights(sh.weight, wlo, whi);
  for (uint32_t first = part.index * static_cast<uint32_t>(part.round); first < a.tokens; first += part.of * static_cast<uint32_t>(part.round)) {
    const int here = static_cast<int>(std::min<uint32_t>(part.round, a.tokens - first));
    const int t = group >> a.log_share[part.w];
    int left = t < here ? part.heads - static_cast<int>(h0) : 0;
    const uint32_t token = first + std::min(t, here - 1), batch = token / a.per_batch, at = token % a.per_batch;
    const T* x = row_of<T>(in, batch, at) + h0 * in.head;
    const T* g = row_of<T>(up, batch, at) + h0 * up.head;
    T* o = row_of<T>(out, batch, at) + h0 * out.head;
    typename L::Raw next = lane.load(x, left > 0), g_next = lane.load(g, given && left > 0);
    __syncthreads();
    stage(a, sh, first, here);
    __syncthreads();
    float cs[kC][kV], sn[kC][kV];
    lane.angles(sh, std::min(t, here - 1) * (a.head_dim / 2), cs, sn);
    for (int base = 0; base < part.heads; base += part.share, left -= part.share, x += x_step, g += g_step, o += o_step) {
      float lo[kC][kV], hi[kC][kV], glo[kC][kV], ghi[kC][kV];
      lane.pairs_of(next, lo, hi);
      lane.pairs_of(g_next, glo, ghi);
      next = lane.load(x + x_step, left > part.share);
      g_next = lane.load(g + g_step, given && left > part.share);
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int i = 0; i < kV; ++i) sum = fmaf(lo[c][i], lo[c][i], fmaf(hi[c][i], hi[c][i], sum));
      const float r = rsqrtf(fmaf(group_sum(sum, a.log_lanes), inv_dim, a.eps));
      float dot = 0.0f;
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          const float ga = glo[c][i], gb = ghi[c][i];
          const float p = fmaf(ga, cs[c][i], gb * sn[c][i]), q = fmaf(gb, cs[c][i], -(ga * sn[c][i]));
          lo[c][i] *= r;
          hi[c][i] *= r;
          if (left > 0) {
            dlo[c][i] = fmaf(p, lo[c][i], dlo[c][i]);
            dhi[c][i] = fmaf(q, hi[c][i], dhi[c][i]);
          }
          glo[c][i] = p * wlo[c][i];
          ghi[c][i] = q * whi[c][i];
          dot = fmaf(glo[c][i], lo[c][i], fmaf(ghi[c][i], hi[c][i], dot));
        }
      dot = group_sum(dot, a.log_lanes) * inv_dim;
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          glo[c][i] = r * fmaf(-lo[c][i], dot, glo[c][i]);
          ghi[c][i] = r * fmaf(-hi[c][i], dot, ghi[c][i]);
        }
      if (left > 0) lane.store(o, glo, ghi);
    }
    if (part.w == 1 && a.dv_out.data != nullptr && t < here) {
      const Heads from = a.dv, to = a.dv_out;
      const T* v = row_of<T>(from, batch, at) + h0 * from.head;
      T* dv = row_of<T>(to, batch, at) + h0 * to.head;
      for (int h = static_cast<int>(h0); h < part.heads; h += part.share, v += part.share * from.head, dv += part.share * to.head) {
        const typename L::Raw raw = lane.load(v, from.data != nullptr);
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          if (!lane.on[c]) continue;
          raw.a[c].store_nt(dv + lane.a[c]);
          raw.b[c].store_nt(dv + lane.b[c]);
        }
      }
    }
  }
  // the workgroup's sums of the weight's gradient: every group's go to LDS, every element is added over the groups by as many lanes as
  // there are, then over those: always in this order
  float* const all = sh.cos;  // and sh.sin behind it: [group][head_dim]
  static_assert(sizeof(sh.cos) + sizeof(sh.sin) >= sizeof(float) * kThreads * 2 * kV * kC && offsetof(Shared, sin) == sizeof(sh.cos), "a lane's sums fit");
  const int groups = kThreads >> a.log_lanes, parts = std::max(1, kThreads / a.head_dim);
  __syncthreads();
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int i = 0; i < kV; ++i)
      if (lane.on[c]) {
        all[group * a.head_dim + lane.element(c, i, false)] = dlo[c][i];
        all[group * a.head_dim + lane.element(c, i, true)] = dhi[c][i];
      }
  __syncthreads();
  for (int i = threadIdx.x; i < parts * a.head_dim; i += kThreads) {
    const int p = i / a.head_dim, d = i - p * a.head_dim;
    float x = 0.0f;
#pragma unroll 4
    for (int q = p; q < groups; q += parts) x += all[q * a.head_dim + d];
    s_dw[i] = x;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.head_dim; d += kThreads) {
    float x = s_dw[d];
    for (int p = 1; p < parts; ++p) x += s_dw[p * a.head_dim + d];
    a.partial[static_cast<int64_t>(blockIdx.x) * a.head_dim + d] = x;
  }
}

// dw = the sum of the workgroups' rows: 64 stretches of rows side by side for 16 columns, then the 64, always in this order.
constexpr int kFoldCols = 16, kFoldRows = 64;
template <typename T>
__global__ __launch_bounds__(kFoldCols* kFoldRows) void qk_rope_fold_kernel(const float* partial, int q_rows, int k_rows, int head_dim, int f32,
                                                                            void* dq_weight, void* dk_weight) {
  __shared__ float s_sum[kFoldRows][kFoldCols];
  const int lane = threadIdx.x % kFoldCols, part = threadIdx.x / kFoldCols;
  const bool is_k = blockIdx.y != 0;
  const int col = static_cast<int>(blockIdx.x) * kFoldCols + lane;
  const int rows = is_k ? k_rows : q_rows;
  if (is_k) partial += static_cast<int64_t>(q_rows) * head_dim;
  float x = 0.0f;
  if (col < head_dim) {
#pragma unroll 16
    for (int r = part; r < rows; r += kFoldRows) x += partial[static_cast<int64_t>(r) * head_dim + col];
  }
  s_sum[part][lane] = x;
  __syncthreads();
  if (part >= 4) return;  // one wave: four sums of 16 each
  x = 0.0f;
#pragma unroll
  for (int p = 0; p < kFoldRows / 4; ++p) x += s_sum[part * (kFoldRows / 4) + p][lane];
  x += __shfl_xor(x, kFoldCols);
  x += __shfl_xor(x, 2 * kFoldCols);
  void* to = is_k ? dk_weight : dq_weight;
  if (part != 0 || col >= head_dim || to == nullptr) return;
  if (f32) static_cast<float*>(to)[col] = x;
  else static_cast<T*>(to)[col] = narrow<T>(x);
}

// ---------------------------------------------------------------- host

int64_t rounds_of(const tdm_qk_shape& s, int round) { return (s.batch * s.tokens + round - 1) / round; }

// How many of a workgroup's groups of lanes share a token, as a power of two: up to eight while at most an eighth of the turns are
// idle (heads that are no multiple), so that a wave's accesses are long; more where there are too few tokens for all workgroups.
int log_share_of(int64_t tokens, int heads, int pairs, int log_groups) {
  auto turns = [&](int log) { return ((heads + (1 << log) - 1) >> log) << log; };
  int log = 0;
  while (log < 3 && log < log_groups && 8 * turns(log + 1) <= 9 * heads) ++log;
  while (log < log_groups && ((1 << (log_groups - log)) > kMostTokens || (1 << (log_groups - log)) * pairs > kLdsPairs || (tokens >> (log_groups - log)) < 512)) ++log;
  return log;
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
  int log_groups = 0;
  while ((kThreads >> a.log_lanes) >> (log_groups + 1) != 0) ++log_groups;
  for (int w = 0; w < 2; ++w) {
    a.log_share[w] = log_share_of(s.batch * s.tokens, a.heads[w], pairs, log_groups);
    a.round[w] = 1 << (log_groups - a.log_share[w]);
    a.groups[w] = a.heads[w] == 0 ? 0u : static_cast<uint32_t>(rounds_of(s, a.round[w]));
  }
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
    const dim3 grid(p.args.groups[0] + p.args.groups[1]);
    require(grid.x < (1u << 24), "qk_norm_rope: 2^24 workgroups or more");
    with_dtype(s.dtype, [&](auto t) {
      using T = decltype(t);
      with_run(p.run, [&](auto v, auto c) {
        if constexpr (v.value * sizeof(T) <= 16) {
          if (p.args.interleaved) hipLaunchKernelGGL((qk_rope_kernel<T, v.value, c.value, true>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), p.args);
          else hipLaunchKernelGGL((qk_rope_kernel<T, v.value, c.value, false>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), p.args);
        }
      });
    });
    check_launch("qk_rope launch");
  });
}

int64_t tdm_k6_qk_norm_rope_grad_workspace(const tdm_qk_shape* shape) {
  int64_t bytes = -1;
  guard([&] {
    check_shape(shape);
    bytes = 2 * std::min<int64_t>(rounds_of(*shape, 1), kMostGroups) * shape->head_dim * 4;
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
    // every workgroup stays for as many rounds as it takes, and leaves one row of partial sums; the workgroups are shared between queries and
    // keys by what they move (of a key's head, the value's copy too)
    const int64_t moved[2] = {3 * int64_t(s.q_heads), (p.args.dv_out.data != nullptr ? 5 : 3) * int64_t(s.kv_heads)};
    for (int w = 0; w < 2 && !nothing; ++w) {
      const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kMostGroups, kGradGroups * moved[w] / (moved[0] + moved[1])));
      p.args.groups[w] = static_cast<uint32_t>(std::min<int64_t>(p.args.groups[w], most));
    }
    const int64_t groups = nothing ? 0 : p.args.groups[0] + p.args.groups[1];
    require(groups == 0 || (workspace != nullptr && workspace_bytes >= groups * s.head_dim * 4 && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
            "qk_norm_rope_grad: the workspace starts on 16 bytes and holds tdm_k6_qk_norm_rope_grad_workspace bytes");
    p.args.partial = static_cast<float*>(workspace);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    with_dtype(s.dtype, [&](auto t) {
      using T = decltype(t);
      if (groups > 0) {
        with_run(p.run, [&](auto v, auto c) {
          if constexpr (v.value * sizeof(T) <= 16) {
            if (p.args.interleaved) hipLaunchKernelGGL((qk_rope_grad_kernel<T, v.value, c.value, true>), dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, st, p.args);
            else hipLaunchKernelGGL((qk_rope_grad_kernel<T, v.value, c.value, false>), dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, st, p.args);
          }
        });
        check_launch("qk_rope_grad launch");
      }
      if (dq_weight != nullptr || dk_weight != nullptr) {
        hipLaunchKernelGGL((qk_rope_fold_kernel<T>), dim3((s.head_dim + kFoldCols - 1) / kFoldCols, 2), dim3(kFoldCols * kFoldRows), 0, st,
                           static_cast<const float*>(workspace), static_cast<int>(p.args.groups[0]), static_cast<int>(p.args.groups[1]), s.head_dim, p.args.weight_f32, dq_weight, dk_weight);
        check_launch("qk_rope_fold launch");
      }
    });
  });
}

}  // extern "C"
