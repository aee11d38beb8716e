// Policy operators on a network's logits rows (include/os_mcts.h, "Policy
// operators"): log probabilities with entropy and top actions, distillation
// from listed targets, and their gradients.
//
// With c = log2(e) / temperature, m the row's maximal logit on a legal action
// and l = log2 sum_i 2^((x_i - m) c), everything follows from (m, l):
//   log2 p_i = (x_i - m) c - l,   H = ln 2 (l - sum_i e_i d_i / sum_i e_i),
// d_i = (x_i - m) c, e_i = 2^d_i; an excluded action is x_i = -inf, e_i = 0.
// Differences come before the scaling, so rows of the type's lowest value or
// with a large common offset lose nothing.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "os_error.h"

namespace osx {
namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;
// d below this is e = 0 in f32 (2^-149 is the least subnormal): keeps 0 * -inf
// out of the entropy's sum.
constexpr float kFloor = -160.0f;
constexpr int kBlock = 256;

struct Rows {
  const void* x;
  const uint8_t* legal;
  int64_t n, ld, lld;
  int32_t v;
  float c;      // log2(e) / temperature
  float inv_t;  // 1 / temperature
};

struct Target {
  const void* ids;
  const void* val;
  int64_t ids_ld, val_ld;
  int32_t k, type, wide;
};

__device__ __forceinline__ float get(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float get(const __bf16* p, int64_t i) { return static_cast<float>(p[i]); }
__device__ __forceinline__ float get(const _Float16* p, int64_t i) { return static_cast<float>(p[i]); }

__device__ __forceinline__ float neg_inf() { return -__builtin_huge_valf(); }

__device__ __forceinline__ int64_t get_id(const void* p, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

template <class T>
__device__ __forceinline__ float logit(const Rows& a, int64_t r, int64_t i) {
  if (a.legal != nullptr && a.legal[r * a.lld + i] == 0) return neg_inf();
  return get(static_cast<const T*>(a.x) + r * a.ld, i);
}

// ln p of a logit: exact for any x the type holds (x - m times c may overflow).
__device__ __forceinline__ float log_p(const Rows& a, float x, float m, float l) {
  return fmaf(x - m, a.inv_t, -l * kLn2);
}

template <class F>
__device__ __forceinline__ float block_fold(float v, float* lds, F f) {
  for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 6); ++w) v = f(v, lds[w]);
  __syncthreads();
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* lds) {
  return block_fold(v, lds, [](float p, float q) { return p + q; });
}
__device__ __forceinline__ float block_max(float v, float* lds) {
  return block_fold(v, lds, [](float p, float q) { return fmaxf(p, q); });
}

// (m, l) of row r, and sum e d / sum e; l and the mean are NaN for a row with a
// NaN or +inf, (0, 0) for an empty one.
template <class T>
__device__ void row_stats(const Rows& a, int64_t r, float* lds, float* m_out, float* l_out,
                          float* mean_out) {
  float m = neg_inf();
  for (int64_t i = threadIdx.x; i < a.v; i += blockDim.x) m = fmaxf(m, logit<T>(a, r, i));
  m = block_max(m, lds);
  if (m == neg_inf()) {  // empty, or only NaN
    m = 0.0f;
  }
  float s = 0.0f, t = 0.0f;
  for (int64_t i = threadIdx.x; i < a.v; i += blockDim.x) {
    const float d = (logit<T>(a, r, i) - m) * a.c;
    const float e = exp2f(d);
    s += e;
    t = fmaf(e, fmaxf(d, kFloor), t);
  }
  s = block_sum(s, lds);
  t = block_sum(t, lds);
  *m_out = m;
  *l_out = s == 0.0f ? 0.0f : log2f(s);
  *mean_out = s == 0.0f ? 0.0f : t / s;
}

// A larger value first, of equal ones the lower index: as unsigned integers.
__device__ __forceinline__ uint64_t top_key(float x, uint32_t i) {
  uint32_t u = __float_as_uint(x + 0.0f);  // -0 and +0 are equal
  u = (u >> 31) ? ~u : (u | 0x80000000u);
  return (static_cast<uint64_t>(u) << 32) | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((u >> 31) ? (u & 0x7FFFFFFFu) : ~u);
}

template <class T>
__global__ __launch_bounds__(kBlock) void k_logprobs(Rows a, const void* actions, int wide,
                                                     float* logprob, float* entropy, float* stats,
                                                     int top, int64_t* top_action,
                                                     float* top_logprob) {
  __shared__ float lds[16];
  __shared__ uint64_t keys[16];
  for (int64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    float m, l, mean;
    row_stats<T>(a, r, lds, &m, &l, &mean);
    if (threadIdx.x == 0) {
      entropy[r] = kLn2 * (l - mean);
      if (stats != nullptr) {
        stats[2 * r] = m;
        stats[2 * r + 1] = l;
      }
      if (actions != nullptr) {
        const int64_t id = get_id(actions, wide, r);
        float v = 0.0f;
        if (id >= a.v) v = __builtin_nanf("");
        else if (id >= 0) v = log_p(a, logit<T>(a, r, id), m, l);
        logprob[r] = v;
      }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < top; ++k) {
      uint64_t best = 0;
      if (l == l)
        for (int64_t i = threadIdx.x; i < a.v; i += blockDim.x) {
          const float x = logit<T>(a, r, i);
          const uint64_t key = top_key(x, static_cast<uint32_t>(i));
          if (x > neg_inf() && key < last && key > best) best = key;
        }
      for (int o = 32; o > 0; o >>= 1) {
        const uint64_t q = __shfl_xor(best, o);
        best = q > best ? q : best;
      }
      if ((threadIdx.x & 63) == 0) keys[threadIdx.x >> 6] = best;
      __syncthreads();
      for (int w = 0; w < kBlock / 64; ++w) best = keys[w] > best ? keys[w] : best;
      __syncthreads();
      last = best;
      if (threadIdx.x == 0) {
        top_action[r * top + k] = best == 0 ? -1 : static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
        top_logprob[r * top + k] =
            l != l ? l : best == 0 ? neg_inf() : log_p(a, key_value(best), m, l);
      }
    }
  }
}

// Writes p_i (f0 + f1 ln p_i) over row r (0 on excluded actions), then the sum
// of the listed entries' weights on top of it where there are any.  entry(j)
// returns (id, weight); id < 0: none.
template <class T, class E>
__device__ void write_grad(const Rows& a, int64_t r, float m, float l, float f0, float f1,
                           T* grad, int k, E entry) {
  auto dense = [&](float x) {
    const float d = (x - m) * a.c - l;
    const float p = exp2f(d);
    return p * fmaf(f1, fmaxf(d, kFloor) * kLn2, f0);
  };
  for (int64_t i = threadIdx.x; i < a.v; i += blockDim.x) {
    const float x = logit<T>(a, r, i);
    grad[i] = static_cast<T>(x == neg_inf() ? 0.0f : dense(x));
  }
  __syncthreads();
  for (int j = threadIdx.x; j < k; j += blockDim.x) {
    const auto e = entry(j);
    if (e.first < 0 || e.first >= a.v) continue;
    const float x = logit<T>(a, r, e.first);
    if (x == neg_inf()) continue;
    float w = 0.0f;
    bool first = true;
    for (int q = 0; q < k; ++q) {
      const auto o = entry(q);
      if (o.first != e.first) continue;
      if (q < j) first = false;
      w += o.second;
    }
    if (first) grad[e.first] = static_cast<T>(dense(x) + w);
  }
  __syncthreads();
}

struct Entry {
  int64_t first;
  float second;
};

template <class T>
__global__ __launch_bounds__(kBlock) void k_logprobs_grad(Rows a, const void* actions, int wide,
                                                          const float* entropy, const float* stats,
                                                          int top, const int64_t* top_action,
                                                          const float* gl, int64_t gls,
                                                          const float* gh, int64_t ghs,
                                                          const float* gt, T* grad,
                                                          int64_t grad_ld) {
  for (int64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    const int64_t id = actions != nullptr && gl != nullptr ? get_id(actions, wide, r) : -1;
    const float g0 = id >= 0 ? gl[r * gls] : 0.0f;
    float sum = id >= a.v ? __builtin_nanf("") : g0;
    for (int k = 0; k < top; ++k)
      if (top_action[r * top + k] >= 0) sum += gt[r * top + k];
    const float h = gh != nullptr ? gh[r * ghs] : 0.0f;
    write_grad<T>(a, r, stats[2 * r], stats[2 * r + 1], -(sum + (h != 0.0f ? h * entropy[r] : 0.0f)) * a.inv_t,
                  -h * a.inv_t, grad + r * grad_ld, top + 1, [&](int j) {
                    if (j == top) return Entry{id, g0 * a.inv_t};
                    return Entry{top_action[r * top + j], gt[r * top + j] * a.inv_t};
                  });
  }
}

// The target's unnormalised value at entry j of row r, relative to `ref`, the
// row's maximum (raw = true: the value itself, -inf: no mass).
__device__ __forceinline__ float target_raw(const Rows& a, const Target& t, int64_t r, int j) {
  if (t.ids != nullptr && get_id(t.ids, t.wide, r * t.ids_ld + j) < 0) return neg_inf();
  const int64_t i = r * t.val_ld + j;
  float z;
  switch (t.type) {
    case OS_AZ_LOGITS_F32: return static_cast<const float*>(t.val)[i];
    case OS_AZ_LOGITS_BF16: return get(static_cast<const __bf16*>(t.val), i);
    case OS_AZ_LOGITS_F16: return get(static_cast<const _Float16*>(t.val), i);
    case OS_AZ_WEIGHTS_F32: z = static_cast<const float*>(t.val)[i]; break;
    default: z = static_cast<float>(static_cast<const int32_t*>(t.val)[i]); break;
  }
  return z <= 0.0f ? neg_inf() : z;
}
__device__ __forceinline__ float target_mass(const Rows& a, const Target& t, float z, float ref) {
  if (z == neg_inf()) return 0.0f;
  return t.type >= OS_AZ_WEIGHTS_F32 ? z / ref : exp2f((z - ref) * a.c);
}

template <class T, bool kGradOnly>
__global__ __launch_bounds__(kBlock) void k_distill(Rows a, Target t, const float* weight,
                                                    int64_t weight_stride, float* loss, float* tent,
                                                    float* stats, T* grad, int64_t grad_ld) {
  __shared__ float lds[16];
  for (int64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    float m, l, mean;
    if (kGradOnly) {
      m = stats[2 * r];
      l = stats[2 * r + 1];
    } else {
      row_stats<T>(a, r, lds, &m, &l, &mean);
    }
    float ref = neg_inf();
    for (int j = threadIdx.x; j < t.k; j += kBlock) ref = fmaxf(ref, target_raw(a, t, r, j));
    ref = block_max(ref, lds);
    if (ref == neg_inf()) ref = 0.0f;
    float tot = 0.0f;
    for (int j = threadIdx.x; j < t.k; j += kBlock)
      tot += target_mass(a, t, target_raw(a, t, r, j), ref);
    tot = block_sum(tot, lds);
    const float inv = tot == 0.0f ? 0.0f : 1.0f / tot;
    float ce = 0.0f, h = 0.0f, bad = 0.0f;
    for (int j = threadIdx.x; j < t.k; j += kBlock) {
      const int64_t id = t.ids != nullptr ? get_id(t.ids, t.wide, r * t.ids_ld + j) : j;
      const float q = target_mass(a, t, target_raw(a, t, r, j), ref) * inv;
      if (id >= a.v) bad = 1.0f;
      else if (id >= 0 && q != 0.0f) ce -= q * log_p(a, logit<T>(a, r, id), m, l);
      if (q != 0.0f) h -= q * (kLn2 * log2f(q));
    }
    ce = block_sum(ce, lds);
    h = block_sum(h, lds);
    bad = block_max(bad, lds);
    if (bad != 0.0f) ce = __builtin_nanf("");
    if (!kGradOnly && threadIdx.x == 0) {
      loss[r] = ce;
      if (tent != nullptr) tent[r] = h;
      if (stats != nullptr) {
        stats[2 * r] = m;
        stats[2 * r + 1] = l;
      }
    }
    if (grad == nullptr) continue;
    const float w = (weight != nullptr ? weight[r * weight_stride] : 1.0f) * a.inv_t;
    const float mass = bad != 0.0f ? __builtin_nanf("") : tot == 0.0f ? 0.0f : tot * inv;
    write_grad<T>(a, r, m, l, w * mass, 0.0f, grad + r * grad_ld, t.k, [&](int j) {
      const int64_t id = t.ids != nullptr ? get_id(t.ids, t.wide, r * t.ids_ld + j) : j;
      return Entry{id, -w * target_mass(a, t, target_raw(a, t, r, j), ref) * inv};
    });
  }
}

// ---- host side ----

int check_rows(const os_az_rows* p, Rows* a) {
  if (!p) return Fail(OS_ERR_INVALID, "null rows");
  if (p->reserved != 0) return Fail(OS_ERR_INVALID, "os_az_rows.reserved must be 0");
  if (p->num_rows < 0 || p->num_actions < 1 || p->ld < 0 || p->legal_ld < 0)
    return Fail(OS_ERR_INVALID, "bad rows shape");
  if (p->num_actions > OS_AZ_MAX_ACTIONS)
    return Fail(OS_ERR_UNSUPPORTED, "more than OS_AZ_MAX_ACTIONS actions");
  if (p->dtype < OS_AZ_F32 || p->dtype > OS_AZ_F16) return Fail(OS_ERR_INVALID, "bad logits dtype");
  // (the scaled differences need a normal, finite 1 / temperature)
  if (!(p->temperature >= 1e-30f && p->temperature <= 1e30f))
    return Fail(OS_ERR_INVALID, "temperature must be in [1e-30, 1e30]");
  const uintptr_t align = p->dtype == OS_AZ_F32 ? 3 : 1;
  if (reinterpret_cast<uintptr_t>(p->logits) & align)
    return Fail(OS_ERR_INVALID, "logits not aligned to their type");
  if (p->num_rows > 0 && !p->logits) return Fail(OS_ERR_INVALID, "null logits");
  *a = Rows{p->logits, p->legal, p->num_rows, p->ld, p->legal_ld, p->num_actions,
            static_cast<float>(1.4426950408889634 / p->temperature),
            static_cast<float>(1.0 / p->temperature)};
  return OS_OK;
}

int check_target(const os_az_target* p, const Rows& a, Target* t) {
  if (!p) return Fail(OS_ERR_INVALID, "null target");
  if (p->reserved != 0) return Fail(OS_ERR_INVALID, "os_az_target.reserved must be 0");
  if (p->k < 0 || p->actions_ld < 0 || p->target_ld < 0)
    return Fail(OS_ERR_INVALID, "bad target shape");
  if (p->k > OS_AZ_MAX_TARGETS)
    return Fail(OS_ERR_UNSUPPORTED, "more than OS_AZ_MAX_TARGETS listed actions");
  if (p->type < OS_AZ_LOGITS_F32 || p->type > OS_AZ_WEIGHTS_I32)
    return Fail(OS_ERR_INVALID, "bad target type");
  if (p->k > 0 && !p->target && a.n > 0) return Fail(OS_ERR_INVALID, "null target values");
  if (p->k > 0 && !p->actions && p->k != a.v && a.n > 0)
    return Fail(OS_ERR_INVALID, "a target without actions needs k = num_actions");
  *t = Target{p->actions, p->target, p->actions_ld, p->target_ld, p->k, p->type, p->wide != 0};
  return OS_OK;
}

int check_grad(const Rows& a, int dtype, const void* grad, int64_t grad_ld) {
  if (grad_ld < a.v) return Fail(OS_ERR_INVALID, "grad_ld < num_actions");
  if (reinterpret_cast<uintptr_t>(grad) & (dtype == OS_AZ_F32 ? 3 : 1))
    return Fail(OS_ERR_INVALID, "grad not aligned to its type");
  return OS_OK;
}

dim3 row_grid(const Rows& a) {
  return dim3(static_cast<unsigned>(std::min<int64_t>(a.n, 1 << 20)));
}

template <class F>
int by_dtype(int dtype, F f) {
  if (dtype == OS_AZ_F32) f(static_cast<float*>(nullptr));
  else if (dtype == OS_AZ_BF16) f(static_cast<__bf16*>(nullptr));
  else f(static_cast<_Float16*>(nullptr));
  HIP_TRY(hipGetLastError());
  return OS_OK;
}

}  // namespace
}  // namespace osx

using namespace osx;

extern "C" {

int64_t os_az_rows_workspace(const os_az_rows* rows, int32_t top) {
  Rows a;
  if (const int rc = check_rows(rows, &a)) return rc;
  if (top < 0 || top > OS_AZ_MAX_TOP) return Fail(OS_ERR_INVALID, "top must be in [0, OS_AZ_MAX_TOP]");
  return 0;
}

int os_az_logprobs_async(const os_az_rows* rows, const void* actions, int32_t wide,
                         float* logprob, float* entropy, float* stats, int32_t top,
                         int64_t* top_action, float* top_logprob, void* workspace,
                         int64_t workspace_bytes, void* hip_stream) {
  Rows a;
  if (const int rc = check_rows(rows, &a)) return rc;
  if (top < 0 || top > OS_AZ_MAX_TOP) return Fail(OS_ERR_INVALID, "top must be in [0, OS_AZ_MAX_TOP]");
  if (a.n == 0) return OS_OK;
  if (!entropy || (top > 0 && (!top_action || !top_logprob)) || (!actions != !logprob))
    return Fail(OS_ERR_INVALID, "null logprobs buffer");
  return by_dtype(rows->dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL(k_logprobs<T>, row_grid(a), dim3(kBlock), 0,
                       static_cast<hipStream_t>(hip_stream), a, actions, wide != 0, logprob,
                       entropy, stats, top, top_action, top_logprob);
  });
}

int os_az_logprobs_grad_async(const os_az_rows* rows, const void* actions, int32_t wide,
                              const float* entropy, const float* stats, int32_t top,
                              const int64_t* top_action, const float* g_logprob,
                              int64_t g_logprob_stride, const float* g_entropy,
                              int64_t g_entropy_stride, const float* g_top, void* grad,
                              int64_t grad_ld, void* hip_stream) {
  Rows a;
  if (const int rc = check_rows(rows, &a)) return rc;
  if (top < 0 || top > OS_AZ_MAX_TOP) return Fail(OS_ERR_INVALID, "top must be in [0, OS_AZ_MAX_TOP]");
  if (g_logprob_stride < 0 || g_entropy_stride < 0) return Fail(OS_ERR_INVALID, "negative stride");
  if (const int rc = check_grad(a, rows->dtype, grad, grad_ld)) return rc;
  if (a.n == 0) return OS_OK;
  if (!stats || !grad || (g_entropy && !entropy) || (g_logprob && !actions))
    return Fail(OS_ERR_INVALID, "null gradient buffer");
  if (!g_top) top = 0;
  if (top > 0 && !top_action) return Fail(OS_ERR_INVALID, "null top_action");
  return by_dtype(rows->dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL(k_logprobs_grad<T>, row_grid(a), dim3(kBlock), 0,
                       static_cast<hipStream_t>(hip_stream), a, actions, wide != 0, entropy, stats,
                       top, top_action, g_logprob, g_logprob_stride, g_entropy, g_entropy_stride,
                       g_top, static_cast<T*>(grad), grad_ld);
  });
}

int os_az_distill_async(const os_az_rows* rows, const os_az_target* target, const float* weight,
                        float* loss, float* target_entropy, float* stats, void* grad,
                        int64_t grad_ld, void* workspace, int64_t workspace_bytes,
                        void* hip_stream) {
  Rows a;
  Target t;
  if (const int rc = check_rows(rows, &a)) return rc;
  if (const int rc = check_target(target, a, &t)) return rc;
  if (grad)
    if (const int rc = check_grad(a, rows->dtype, grad, grad_ld)) return rc;
  if (a.n == 0) return OS_OK;
  if (!loss) return Fail(OS_ERR_INVALID, "null loss");
  return by_dtype(rows->dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL((k_distill<T, false>), row_grid(a), dim3(kBlock), 0,
                       static_cast<hipStream_t>(hip_stream), a, t, weight, int64_t{1}, loss,
                       target_entropy, stats, static_cast<T*>(grad), grad_ld);
  });
}

int os_az_distill_grad_async(const os_az_rows* rows, const os_az_target* target,
                             const float* weight, int64_t weight_stride, const float* stats,
                             void* grad, int64_t grad_ld, void* hip_stream) {
  Rows a;
  Target t;
  if (const int rc = check_rows(rows, &a)) return rc;
  if (const int rc = check_target(target, a, &t)) return rc;
  if (weight_stride < 0) return Fail(OS_ERR_INVALID, "negative stride");
  if (const int rc = check_grad(a, rows->dtype, grad, grad_ld)) return rc;
  if (a.n == 0) return OS_OK;
  if (!stats || !grad) return Fail(OS_ERR_INVALID, "null gradient buffer");
  return by_dtype(rows->dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL((k_distill<T, true>), row_grid(a), dim3(kBlock), 0,
                       static_cast<hipStream_t>(hip_stream), a, t, weight, weight_stride,
                       static_cast<float*>(nullptr), static_cast<float*>(nullptr),
                       const_cast<float*>(stats), static_cast<T*>(grad), grad_ld);
  });
}

}  // extern "C"
