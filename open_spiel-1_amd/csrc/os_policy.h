// Policy operators on a network's logits rows (include/os_mcts.h, "Policy
// operators"): log probabilities with entropy and top actions, distillation
// from listed targets, and their gradients.  Kernels; os_policy.hip checks the
// arguments and chooses among them, os_policy_{f32,bf16,f16}.hip instantiate
// them, one unit a type so that they build in parallel.
//
// Mathematics.  With c = log2(e) / temperature, m the row's maximal logit on an
// allowed action and l = log2 sum_i 2^((x_i - m) c), everything follows from
// (m, l): log2 p_i = (x_i - m) c - l, and with d_i = (x_i - m) c, e_i = 2^d_i
// the entropy is ln 2 (l - sum e_i d_i / sum e_i).  An excluded action is
// x_i = -inf, e_i = 0.  The difference is taken before the scaling, so rows of
// the type's lowest value, or with a large common offset, lose nothing; sums
// are held in float32, at most 128 terms a lane, then joined in trees.
//
// What bounds it.  Two to four bytes an element against one exponential and
// some eight other operations (two exponentials with the gradient): HBM, when
// the card is full, with the vector units about half busy - so each row is read
// ONCE, by whole workgroups, and stays in registers (16 chunks of 16 bytes a
// lane: up to 256 KiB a workgroup, the register file being 512 KiB a compute
// unit) from the sums to the gradient or the selection of the top actions.
// 2048 rows of 131072 bf16 actions: top 20 in 123 us (4.4 TB/s read), loss and
// gradient in 244 us (4.4 TB/s read and written; a copy of 2 GiB: 4.9 TB/s).
// Short rows (k_wave) are bound by the vector units, few rows by latency.
// The maximum and the sums run together over the chunks as they arrive (a
// running maximum, the sums rescaled by it), and a chunk's registers are
// reloaded with the next row's data as soon as the last pass is through with
// them, so the loads of row r + 1 run under the arithmetic of row r.
#ifndef OS_POLICY_H_
#define OS_POLICY_H_

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/os_mcts.h"

namespace osp {

constexpr float kLn2 = 0.69314718055994530942f;
// 2^d is 0 here (the exponential keeps no subnormals: from -126 down): keeps
// 0 * -inf out of the sums.
constexpr float kFloor = -160.0f;
// Rows whose maximum times c is further out than this ("wild") take the plain
// form 2^((x - m) c): beyond it the rounding of m c alone would be over half a
// unit of the exponent.
constexpr float kWild = 16777216.0f;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr int kTinyMax = 64;       // rows of up to this many actions: 16 lanes each
constexpr int kMaxWaves = 16;
constexpr int kMaxSplit = 64;      // parts of a row
constexpr int kCandidates = 512;   // top actions: LDS list
constexpr int kWaveCandidates = 192;  // of a wave alone (a multiple of 64)
constexpr int kWaveMax = 2048;     // of up to this many: a wave each, 32 actions a lane
constexpr int kFewChunks = 4;      // chunks a lane of k_rows: the least,
constexpr int kMidChunks = 8;      // the most with a mask
constexpr int kChunks = 16;        // and without

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

// How the workgroups share the rows: blockIdx.y is a part of a row, `part`
// actions long (a multiple of 64; the last part is shorter, never below 64
// where there are several), blockIdx.x strides over the rows.
struct Parts {
  int32_t parts, part;
};

// One part's sums, for k_join; its top keys follow in a list of their own.
struct PartSums {
  float m, s, t, pad;
};

struct LogprobArgs {
  const void* actions;
  int32_t wide, top;
  float* logprob;
  float* entropy;
  float* stats;
  int64_t* top_action;
  float* top_logprob;
  PartSums* sums;      // != nullptr: write parts, not results
  uint64_t* part_keys;
};

struct LogprobGradArgs {
  const void* actions;
  int32_t wide, top;
  const float* entropy;
  const float* stats;
  const int64_t* top_action;
  const float* gl;
  int64_t gls;
  const float* gh;
  int64_t ghs;
  const float* gt;
  void* grad;
  int64_t grad_ld;
};

struct DistillArgs {
  Target t;
  const float* weight;
  int64_t weight_stride;
  float* loss;
  float* tent;
  float* stats;  // kDistillGrad reads them
  void* grad;
  int64_t grad_ld;
  int32_t hash;  // LDS table entries (a power of two)
};

struct JoinArgs {
  LogprobArgs lp;
  DistillArgs ds;
  int32_t parts;
};

enum Op : int { kLogprobs, kLogprobsTop, kLogprobsGrad, kDistill, kDistillFused, kDistillGrad };

// The compiler must take x for a new value: it would otherwise keep what was
// computed from it earlier (every chunk's converted elements, every offset) in
// registers that the rows need.  No instruction.
template <class V>
__device__ __forceinline__ void renew(V& x) {
  asm volatile("" : "+v"(x));
}
__device__ __forceinline__ int renewed_scalar(int x) {
  asm volatile("" : "+s"(x));
  return x;
}

__device__ __forceinline__ float neg_inf() { return -__builtin_huge_valf(); }
__device__ __forceinline__ float exp2_(float d) { return __builtin_amdgcn_exp2f(d); }

// ---- element types ----

template <class T>
constexpr int kPer = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte chunk

using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using f32x2 = __attribute__((ext_vector_type(2))) float;

__device__ __forceinline__ float get(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float get(const __bf16* p, int64_t i) { return static_cast<float>(p[i]); }
__device__ __forceinline__ float get(const _Float16* p, int64_t i) { return static_cast<float>(p[i]); }

// Rows start anywhere their type may (an odd row stride, a view's column
// offset): wide accesses are declared with the element's alignment only.
// kStream: read or written once (a hint to the caches).
template <bool kStream, class T, class W>
__device__ __forceinline__ W load_at(const T* p) {
  typedef W Any __attribute__((aligned(sizeof(T))));
  if constexpr (kStream) return __builtin_nontemporal_load(reinterpret_cast<const Any*>(p));
  else return *reinterpret_cast<const Any*>(p);
}
template <bool kStream, class T, class W>
__device__ __forceinline__ void store_at(T* p, W w) {
  typedef W Any __attribute__((aligned(sizeof(T))));
  if constexpr (kStream) __builtin_nontemporal_store(w, reinterpret_cast<Any*>(p));
  else *reinterpret_cast<Any*>(p) = w;
}

// A chunk's mask bytes.
template <int kE>
struct __attribute__((packed, aligned(1))) MaskWord {
  uint32_t w[kE / 4];
  __device__ __forceinline__ bool allows(int j) const {
    return static_cast<uint8_t>(w[j / 4] >> (8 * (j % 4))) != 0;
  }
};
template <>
struct __attribute__((packed, aligned(1))) MaskWord<2> {
  uint16_t w;
  __device__ __forceinline__ bool allows(int j) const { return (w & (0xFFu << (8 * j))) != 0; }
};

// A chunk of kE elements: W is u32x4, or u32x2 (k_wave).
template <class T, class W, int kE>
__device__ __forceinline__ void unpack(W r, float (&x)[kE]) {
  static_assert(sizeof(W) == kE * sizeof(T));
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int j = 0; j < kE; ++j) x[j] = __uint_as_float(r[j]);
  } else if constexpr (std::is_same_v<T, __bf16>) {
#pragma unroll
    for (int j = 0; j < kE / 2; ++j) {
      x[2 * j] = __uint_as_float(r[j] << 16);
      x[2 * j + 1] = __uint_as_float(r[j] & 0xFFFF0000u);
    }
  } else {
    using h2 = __attribute__((ext_vector_type(2))) _Float16;
#pragma unroll
    for (int j = 0; j < kE / 2; ++j) {
      const h2 h = __builtin_bit_cast(h2, static_cast<uint32_t>(r[j]));
      x[2 * j] = static_cast<float>(h[0]);
      x[2 * j + 1] = static_cast<float>(h[1]);
    }
  }
}
// Round to nearest even, once.
template <class T, class W, int kE>
__device__ __forceinline__ W pack(const float (&x)[kE]) {
  static_assert(sizeof(W) == kE * sizeof(T));
  W r;
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int j = 0; j < kE; ++j) r[j] = __float_as_uint(x[j]);
  } else {
    using h2 = __attribute__((ext_vector_type(2))) T;
#pragma unroll
    for (int j = 0; j < kE / 2; ++j) {
      const f32x2 f = {x[2 * j], x[2 * j + 1]};
      r[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, h2));
    }
  }
  return r;
}

// A load at a uniform address of memory that the kernel does not write: on the
// scalar unit, in a queue of its own (vector loads come back in order, so one
// for a single value would wait for the whole next row's).
template <class V>
__device__ __forceinline__ V uniform(const V* p, int64_t i) {
  return reinterpret_cast<const __attribute__((address_space(4))) V*>(
      reinterpret_cast<uintptr_t>(p))[i];
}
__device__ __forceinline__ int64_t uniform_id(const void* p, int wide, int64_t i) {
  return wide ? uniform(static_cast<const int64_t*>(p), i)
              : uniform(static_cast<const int32_t*>(p), i);
}
__device__ __forceinline__ int64_t get_id(const void* p, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// One element of row r (-inf: excluded).
template <class T>
__device__ __forceinline__ float logit(const Rows& a, int64_t r, int64_t i) {
  const float x = get(static_cast<const T*>(a.x) + r * a.ld, i);
  return a.legal != nullptr && a.legal[r * a.lld + i] == 0 ? neg_inf() : x;
}

// ln p of a logit: right for any x of the type ((x - m) c may overflow, and x - m
// where the temperature brings it back: hence the halves).
__device__ __forceinline__ float log_p(const Rows& a, float x, float m, float l) {
  return fmaf(0.5f * x - 0.5f * m, 2.0f * a.inv_t, -l * kLn2);
}

// The largest of a chunk's values: v_maximum3_f32, which needs no quieting of
// its operands (a NaN passes through: callers take it for none).
template <int kE>
__device__ __forceinline__ float largest(const float (&x)[kE]) {
  const auto mx = [](float p, float q) { return __builtin_elementwise_maximum(p, q); };
  float m = mx(mx(x[0], x[1]), x[2]);
#pragma unroll
  for (int j = 3; j + 1 < kE; j += 2) m = mx(mx(m, x[j]), x[j + 1]);
  return mx(m, x[kE - 1]);
}

// ---- reductions ----

template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xF, 0xF, true));
}
template <int kCtrl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xF, 0xF, true));
}
struct Add {
  __device__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct MinU {
  __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a < b ? a : b; }
};
// Over each 16 lanes (pairs, quads, then mirrored halves): all of them get it.
template <class T, class F>
__device__ __forceinline__ T fold16(T v, F f) {
  v = f(v, dpp<0xB1>(v));
  v = f(v, dpp<0x4E>(v));
  v = f(v, dpp<0x141>(v));
  return f(v, dpp<0x140>(v));
}
__device__ __forceinline__ float lane_at(float v, int i) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
}
// Over the wave: within rows of 16 lanes as above, then row 0 into 1 and 2 into
// 3, then both into the last row; a uniform result.  Written out because the
// compiler quiets both operands of every maximum (three instructions a step for
// one).  A DPP operand needs two wait states after its write: the s_nop.
#define OSP_FOLD64(op)                                                    \
  "s_nop 1\n"                                                             \
  op " %0, %1, %1 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"       \
  "s_nop 1\n"                                                             \
  op " %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"       \
  "s_nop 1\n"                                                             \
  op " %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n"           \
  "s_nop 1\n"                                                             \
  op " %0, %0, %0 row_mirror row_mask:0xf bank_mask:0xf\n"                \
  "s_nop 1\n"                                                             \
  op " %0, %0, %0 row_bcast:15 row_mask:0xa bank_mask:0xf\n"              \
  "s_nop 1\n"                                                             \
  op " %0, %0, %0 row_bcast:31 row_mask:0xc bank_mask:0xf\n"              \
  "s_nop 1\n"
__device__ __forceinline__ float fold64(float v, Max) {
  float r;
  asm volatile(OSP_FOLD64("v_max_f32_dpp") : "=&v"(r) : "v"(v));
  return lane_at(r, 63);
}
__device__ __forceinline__ float fold64(float v, Add) {
  float r;
  asm volatile(OSP_FOLD64("v_add_f32_dpp") : "=&v"(r) : "v"(v));
  return lane_at(r, 63);
}
#undef OSP_FOLD64

// Sums relative to a maximum (-inf: none): s = sum 2^((x - m) c), t = sum of
// that times (x - m) c.
struct Sums {
  float m, s, t;
};
template <bool kEnt>
__device__ __forceinline__ Sums fold_sums(Sums a, float c) {
  Sums r;
  r.m = fold64(a.m, Max{});
  const float d = (a.m - (r.m == neg_inf() ? 0.0f : r.m)) * c;
  const float f = exp2_(d);
  r.s = fold64(a.s * f, Add{});
  r.t = kEnt ? fold64(f * fmaf(a.s, fmaxf(d, kFloor), a.t), Add{}) : 0.0f;
  return r;
}

// A target's unnormalised mass is relative to a reference, the row's largest
// value: logits 2^((z - ref) c), weights z times the power of two that brings
// the reference near 1 (sums neither overflow nor vanish, and no division an
// entry).  An entry without mass has the value 0 (weights) or -inf (logits).
__device__ __forceinline__ bool is_weights(const Target& t) { return t.type >= OS_AZ_WEIGHTS_F32; }
__device__ __forceinline__ float no_mass(const Target& t) { return is_weights(t) ? 0.0f : neg_inf(); }
__device__ __forceinline__ int weight_scale_bits(float ref) {
  return max(0x7E800000 - (__float_as_int(ref) & 0x7F800000), 0x00800000);
}
__device__ __forceinline__ float target_mass(const Target& t, float c, float z, float ref) {
  if (is_weights(t)) return z * __int_as_float(weight_scale_bits(ref));
  return exp2_((z - (ref == neg_inf() ? 0.0f : ref)) * c);
}
// What takes a mass relative to `from` to one relative to `to`, not below it.
__device__ __forceinline__ float mass_step(const Target& t, float c, float from, float to) {
  if (is_weights(t)) {
    const int b = 0x3F800000 + weight_scale_bits(to) - weight_scale_bits(from);
    return b <= 0 ? 0.0f : __int_as_float(b);
  }
  return from == to ? 1.0f : exp2_((from - to) * c);
}
// A mass's share of the total, inv = 1 / total (0: no mass): the quotient with one
// correction, so that a target with all its mass in one place has q = 1 there and
// an entropy of 0.
__device__ __forceinline__ float share(float mass, float total, float inv) {
  const float q = mass * inv;
  return fmaf(fmaf(-q, total, mass), inv, q);
}
// Sums taken with d = x c - R, R = m c rounded, hold e0 = 2^off, off = m c - R,
// where those relative to m hold 1: s becomes share(s, e0, ..), never below 1, and
// t = sum e d becomes e0 times sum e (x - m) c: the maximum's own e0 off goes as it
// came, off times the others' sum with it.  So a row's only action has s = 1, t = 0
// and a log probability and entropy of exactly 0, and no log probability is above 0
// (2^-off as a factor instead: up to 6e-8 off either way).
__device__ __forceinline__ float mean_part(float s, float t, float e0, float off) {
  return fmaf(-off, s - e0, t - e0 * off);
}
// ln q of a mass share.
__device__ __forceinline__ float log_share(float q) {
  return kLn2 * fmaxf(__builtin_amdgcn_logf(q), kFloor);
}
__device__ __forceinline__ float target_value(const Target& t, int64_t i) {
  float z;
  switch (t.type) {
    case OS_AZ_LOGITS_F32: return static_cast<const float*>(t.val)[i];
    case OS_AZ_LOGITS_BF16: return get(static_cast<const __bf16*>(t.val), i);
    case OS_AZ_LOGITS_F16: return get(static_cast<const _Float16*>(t.val), i);
    case OS_AZ_WEIGHTS_F32: z = static_cast<const float*>(t.val)[i]; break;
    default: z = static_cast<float>(static_cast<const int32_t*>(t.val)[i]); break;
  }
  return z <= 0.0f ? 0.0f : z;
}
// Entry j of a row: its action (< 0: none) and value.
struct Entry {
  int64_t id;
  float z;
};
__device__ __forceinline__ Entry target_entry(const Target& t, int64_t r, int j) {
  Entry e;
  e.id = t.ids != nullptr ? get_id(t.ids, t.wide, r * t.ids_ld + j) : j;
  e.z = e.id < 0 ? no_mass(t) : target_value(t, r * t.val_ld + j);
  return e;
}
// Entries first, first + step, .. of a row (those below k; the others none):
// every load is issued before one is waited for, and all are waited for here.
// id -1: none or past the v actions (then bad); z: the value, no_mass() where
// there is none.
template <int kCount>
__device__ __forceinline__ void target_entries(const Target& t, int64_t r, int first, int step,
                                               int v, int (&id)[kCount], float (&z)[kCount],
                                               float& bad) {
#pragma unroll
  for (int i = 0; i < kCount; ++i) {
    id[i] = -1;
    z[i] = no_mass(t);
  }
  if (t.k == 0) return;
  // (uniform: how many of the batches hold any entry)
  const int rounds = min(kCount, (t.k + step - 1) / step);
  const auto at = [&](int i) { return min(first + i * step, t.k - 1); };
  const auto all = [&](auto f) {
#pragma unroll
    for (int i = 0; i < kCount; ++i)
      if (i < rounds) f(i);
  };
  int raw[kCount];  // (of an int64 only whether it is below 0 or past the actions counts)
  if (t.ids == nullptr) {
    all([&](int i) { raw[i] = at(i); });
  } else if (t.wide) {
    const int64_t* const p = static_cast<const int64_t*>(t.ids) + r * t.ids_ld;
    int64_t wide[kCount];
    all([&](int i) { wide[i] = p[at(i)]; });
    all([&](int i) {
      raw[i] = static_cast<int>(wide[i] < 0 ? -1 : wide[i] < v ? wide[i] : int64_t{v});
    });
  } else {
    const int32_t* const p = static_cast<const int32_t*>(t.ids) + r * t.ids_ld;
    all([&](int i) { raw[i] = p[at(i)]; });
  }
  const auto values = [&](auto* p) {
    p += r * t.val_ld;
    all([&](int i) { z[i] = static_cast<float>(p[at(i)]); });
  };
  switch (t.type) {
    case OS_AZ_LOGITS_F32:
    case OS_AZ_WEIGHTS_F32: values(static_cast<const float*>(t.val)); break;
    case OS_AZ_LOGITS_BF16: values(static_cast<const __bf16*>(t.val)); break;
    case OS_AZ_LOGITS_F16: values(static_cast<const _Float16*>(t.val)); break;
    default: values(static_cast<const int32_t*>(t.val)); break;
  }
  all([&](int i) {
    // (selects only: written with && and an if, the compiler of ROCm 7.2 lost the
    // weights' z <= 0 case)
    const bool in = (first + i * step < t.k) & (raw[i] >= 0), past = raw[i] >= v;
    const bool none = !in | (is_weights(t) & (z[i] <= 0.0f));
    bad = (in & past) ? 1.0f : bad;
    id[i] = (in & !past) ? raw[i] : -1;
    z[i] = none ? no_mass(t) : z[i];
  });
}
// The same in two halves, as they lie in memory in between: load() issues every
// load and finish() is the first to wait for one.  (Held across a row by k_rows.
// k_wave's six entries a lane, held across the sums in this form, spill: 16384 x
// 362 visit counts 33 -> 43 us.)
template <int kCount>
struct RawEntries {
  int64_t id[kCount];
  uint32_t z[kCount];

  // (uniform: how many of the batches hold any entry)
  __device__ __forceinline__ static int rounds(const Target& t, int step) {
    return min(kCount, (t.k + step - 1) / step);
  }
  __device__ __forceinline__ void load(const Target& t, int64_t r, int first, int step) {
    if (t.k == 0) return;
    const int n = rounds(t, step);
    const auto all = [&](auto f) {
#pragma unroll
      for (int i = 0; i < kCount; ++i)
        if (i < n) f(i, min(first + i * step, t.k - 1));
    };
    if (t.ids == nullptr) {
      all([&](int i, int j) { id[i] = j; });
    } else if (t.wide) {
      const int64_t* const p = static_cast<const int64_t*>(t.ids) + r * t.ids_ld;
      all([&](int i, int j) { id[i] = p[j]; });
    } else {
      const int32_t* const p = static_cast<const int32_t*>(t.ids) + r * t.ids_ld;
      all([&](int i, int j) { id[i] = static_cast<uint32_t>(p[j]); });
    }
    if (t.type == OS_AZ_LOGITS_BF16 || t.type == OS_AZ_LOGITS_F16) {
      const uint16_t* const p = static_cast<const uint16_t*>(t.val) + r * t.val_ld;
      all([&](int i, int j) { z[i] = p[j]; });
    } else {
      const uint32_t* const p = static_cast<const uint32_t*>(t.val) + r * t.val_ld;
      all([&](int i, int j) { z[i] = p[j]; });
    }
  }
  // id -1: none or past the v actions (then bad); z: the value, no_mass() where
  // there is none.
  __device__ __forceinline__ void finish(const Target& t, int first, int step, int v,
                                         int (&out)[kCount], float (&value)[kCount],
                                         float& bad) const {
    const int n = rounds(t, step);
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      out[i] = -1;
      value[i] = no_mass(t);
      if (i < n) {
        float f = __uint_as_float(z[i]);
        if (t.type == OS_AZ_LOGITS_BF16) f = __uint_as_float(z[i] << 16);
        else if (t.type == OS_AZ_LOGITS_F16)
          f = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(z[i])));
        else if (t.type == OS_AZ_WEIGHTS_I32) f = static_cast<float>(static_cast<int32_t>(z[i]));
        // (a 32-bit action's sign is found here, not before its load is waited for)
        const int64_t a = t.ids != nullptr && !t.wide ? static_cast<int32_t>(id[i]) : id[i];
        // (selects only: written with && and an if, the compiler of ROCm 7.2
        // lost the weights' f <= 0 case)
        const bool in = (first + i * step < t.k) & (a >= 0), past = a >= v;
        const bool none = !in | (is_weights(t) & (f <= 0.0f));
        bad = (in & past) ? 1.0f : bad;
        out[i] = (in & !past) ? static_cast<int>(a) : -1;
        value[i] = none ? no_mass(t) : f;
      }
    }
  }
};
// Running (maximum, mass relative to it) of target entries.
struct Mass {
  float z, s;
};
__device__ __forceinline__ void mass_add(const Target& t, float c, float z, Mass& a) {
  const float to = fmaxf(a.z, z);
  a.s = fmaf(a.s, mass_step(t, c, a.z, to), target_mass(t, c, z, to));
  a.z = to;
}
template <int kCount>
__device__ __forceinline__ Mass mass_of(const Target& t, float c, const float (&z)[kCount]) {
  Mass a{z[0], 0.0f};
#pragma unroll
  for (int i = 1; i < kCount; ++i) a.z = fmaxf(a.z, z[i]);
#pragma unroll
  for (int i = 0; i < kCount; ++i) a.s += target_mass(t, c, z[i], a.z);
  return a;
}
template <class MaxF, class AddF>
__device__ __forceinline__ Mass mass_fold(const Target& t, float c, Mass a, MaxF maxf, AddF addf) {
  const float z = maxf(a.z);
  return Mass{z, addf(a.s * mass_step(t, c, a.z, z))};
}

// ---- top actions ----

// A larger value first, of equal ones the lower index, as unsigned integers; 0
// is no key.
__device__ __forceinline__ uint64_t top_key(float x, uint32_t i) {
  uint32_t u = __float_as_uint(x + 0.0f);  // -0 and +0 are equal
  u = (u >> 31) ? ~u : (u | 0x80000000u);
  return (static_cast<uint64_t>(u) << 32) | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((u >> 31) ? (u & 0x7FFFFFFFu) : ~u);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) {
  return 0xFFFFFFFFu - static_cast<uint32_t>(k);
}
__device__ __forceinline__ uint64_t fold64_max(uint64_t v) {
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t q = __shfl_xor(v, o);
    v = q > v ? q : v;
  }
  return v;
}
// One of the lanes' values with at least k of them at or above it, and usually
// few more (-inf where fewer than k lanes hold any): a bound of the k-th largest
// element from below.  Bisection between the least and the largest (`most`) over
// 2^16 steps, counting with ballots on the scalar unit: six rounds or so of one
// vector operation, where ranking every lane against every other takes 192.
__device__ __forceinline__ float kth_bound(float v, float most, int k) {
  if (k == 1) return most;
  const float inf = __builtin_huge_valf();
  const bool any = v > neg_inf();
  if (__builtin_popcountll(__ballot(any)) < k) return neg_inf();
  // (halves: the difference of two finite values is finite)
  const float least = -0.5f * fold64(any ? -v : -inf, Max{});
  const float scale = 65535.0f * __builtin_amdgcn_rcpf(fmaf(most, 0.5f, -least));
  const int q = any ? static_cast<int>(fminf(fmaf(v, 0.5f, -least) * scale, 65535.0f)) : -1;
  const int enough = k + (k >> 2) + 3;
  int lo = 0, hi = 65536;
#pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    const int n = __builtin_popcountll(__ballot(q >= mid));
    if (n >= k) lo = mid;
    else hi = mid;
    if (n >= k && n <= enough) break;
  }
  return -fold64(q >= lo ? -v : -inf, Max{});
}

// The k-th largest (k >= 1) of one key a lane.
__device__ __forceinline__ uint64_t kth64(uint64_t key, int k) {
  const int lane = threadIdx.x & 63;
  const uint32_t lo = static_cast<uint32_t>(key), hi = static_cast<uint32_t>(key >> 32);
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j < 64; ++j) {
    const uint64_t q =
        (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(hi), j))) << 32) |
        static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(lo), j));
    rank += q > key || (q == key && j < lane) ? 1 : 0;
  }
  const uint64_t at = __ballot(rank == k - 1);
  const int src = __builtin_ctzll(at);
  return (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(hi), src))) << 32) |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(lo), src));
}

struct Found {
  float x;
  int i;
};
struct TopLds {
  uint64_t group[64];  // largest key of lane i of every wave
  float bound;         // what the top-th largest is not below,
  int cut;             // and, at the bound, where the last needed one's chunk ends
  uint32_t chunks, count;
  int chunk[kCandidates];  // starts of the chunks that reach the bound
  uint64_t cand[kCandidates];
};

// ---- the listed entries of a gradient ----

// A row's listed actions in an open-addressed LDS table: key (action, -1:
// free), the weight to add there and its logit.  Distinct actions are inserted
// in parallel; where one is met twice, `twice` is set and one lane rebuilds the
// table in list order, so a sum never depends on the order of waves.
struct Table {
  int32_t* key;
  float* w;
  float* x;
  int32_t mask;
};
__device__ __forceinline__ uint32_t table_slot(const Table& t, int32_t id) {
  return (static_cast<uint32_t>(id) * 2654435761u >> 16) & t.mask;
}
__device__ __forceinline__ void table_clear(const Table& t, int tid, int step) {
  for (int i = tid; i <= t.mask; i += step) t.key[i] = -1;
}
__device__ __forceinline__ bool table_put(const Table& t, int32_t id, float w, float x) {
  uint32_t s = table_slot(t, id);
  for (;;) {  // (at most half full: a free slot is met)
    const int32_t old = atomicCAS(&t.key[s], -1, id);
    if (old == -1) {
      t.w[s] = w;
      t.x[s] = x;
      return true;
    }
    if (old == id) return false;
    s = (s + 1) & t.mask;
  }
}
// One lane alone: adds to what is there.
__device__ __forceinline__ void table_add(const Table& t, int32_t id, float w, float x) {
  uint32_t s = table_slot(t, id);
  while (t.key[s] != -1 && t.key[s] != id) s = (s + 1) & t.mask;
  if (t.key[s] == id) {
    t.w[s] += w;
  } else {
    t.key[s] = id;
    t.w[s] = w;
    t.x[s] = x;
  }
}

// p_i (f0 + f1 log2 p_i) of a logit x, as e (g0 + g1 d) with d = x c - R in one
// operation, e = 2^d and R = m c rounded: what the rounding leaves out and l are
// in g0 and g1.  A wild row takes d = (x - m) c, and so does one whose l is 0 (its
// only action, or one that leaves the others nothing, then has p = 1 and a
// gradient of exactly 0) and every row with kFar.
template <bool kFar>
struct Dense {
  float c, ref, m, g0, g1;
  bool far;    // d = (x - m) c
  bool plain;  // neither far nor with a factor that is not finite
  __device__ __forceinline__ Dense(float m_, float l, float c_, float f0, float f1)
      : c(c_), ref(m_ * c_), m(m_) {
    far = kFar || l == 0.0f || !(fabsf(ref) <= kWild);
    const float k = (far ? 0.0f : fmaf(-m, c, ref)) - l;
    const float f = exp2_(k);
    g0 = fmaf(f1, k, f0) * f;
    g1 = f1 * f;
    const float inf = __builtin_huge_valf();
    plain = !far && fabsf(g0) < inf && fabsf(g1) < inf;
  }
  template <bool kLog>
  __device__ __forceinline__ float scaled(float d) const {
    const float e = exp2_(d);
    return kLog ? e * fmaf(g1, fmaxf(d, kFloor), g0) : e * g0;
  }
  // plain rows
  template <bool kLog>
  __device__ __forceinline__ float at(float x) const {
    return scaled<kLog>(fmaf(x, c, -ref));
  }
  // any row: an excluded action's is 0 whatever the factors
  template <bool kLog>
  __device__ __forceinline__ float any(float x) const {
    if (x == neg_inf()) return 0.0f;
    return scaled<kLog>(kFar || far ? (x - m) * c : fmaf(x, c, -ref));
  }
};

// ---- a row's single values ----

template <int kOp>
using ArgsOf = std::conditional_t<kOp == kLogprobs || kOp == kLogprobsTop, LogprobArgs,
                                  std::conditional_t<kOp == kLogprobsGrad, LogprobGradArgs, DistillArgs>>;

// Fetched a row ahead: a scalar load waited for where it is used would cost its
// whole latency at the start of every row.
template <int kOp>
struct RowValues {
  int64_t given;  // kLogprobs*: the given action, -1: none
  float m, l;     // kLogprobsGrad, kDistillGrad: the stats
  float gl, gh, entropy, weight;

  __device__ __forceinline__ static RowValues at(const ArgsOf<kOp>& g, int64_t r) {
    RowValues v{-1, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 1.0f};
    if constexpr (kOp == kLogprobs || kOp == kLogprobsTop || kOp == kLogprobsGrad)
      if (g.actions != nullptr) v.given = uniform_id(g.actions, g.wide, r);
    if constexpr (kOp == kLogprobsGrad || kOp == kDistillGrad) {
      v.m = uniform(g.stats, 2 * r);
      v.l = uniform(g.stats, 2 * r + 1);
    }
    if constexpr (kOp == kLogprobsGrad) {
      if (g.gl != nullptr) v.gl = uniform(g.gl, r * g.gls);
      if (g.gh != nullptr) {
        v.gh = uniform(g.gh, r * g.ghs);
        v.entropy = uniform(g.entropy, r);
      }
    }
    if constexpr (kOp == kDistillFused || kOp == kDistillGrad)
      if (g.weight != nullptr) v.weight = uniform(g.weight, r * g.weight_stride);
    return v;
  }
};

// ---- long rows ----

// One workgroup of `nw` waves a row (or a part of one), kN chunks of 16 bytes a
// lane: kFewChunks where there are few rows (more waves each), kMidChunks or
// kChunks where there are many; with a mask, whose bytes want registers too, at
// most kMidChunks.
// kStream: the logits exceed the last-level cache, so nothing of them is worth
// keeping there (131072 bf16 actions x 2048 rows, 64 targets: 268 -> 253 us).
template <class T, bool kMask, int kN, int kOp, bool kStream>
__global__ __launch_bounds__(64 * kMaxWaves) void k_rows(Rows a, Parts pt, ArgsOf<kOp> g) {
  constexpr int kE = kPer<T>;
  constexpr bool kSums = kOp != kLogprobsGrad && kOp != kDistillGrad;
  constexpr bool kGrad = kOp == kLogprobsGrad || kOp == kDistillGrad || kOp == kDistillFused;
  constexpr bool kTop = kOp == kLogprobsTop;
  constexpr bool kEnt = kOp == kLogprobs || kOp == kLogprobsTop;
  constexpr bool kTarget = kOp == kDistill || kOp == kDistillFused || kOp == kDistillGrad;
  constexpr bool kSecond = kGrad;                    // a second pass over the registers
  constexpr int kHeld = kN == kFewChunks ? 4 : 1;    // target entries a lane keeps
  using Word = MaskWord<kE>;
  extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];
  __shared__ float red[2][kMaxWaves][8];
  __shared__ float red2[2][kMaxWaves][2];
  __shared__ int twice[2];
  __shared__ std::conditional_t<kTop, TopLds, int> top_lds;

  const int bd = blockDim.x, tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = bd >> 6;
  const int lo = blockIdx.y * pt.part;
  const int len = min(pt.part, a.v - lo);
  const T* const xb = static_cast<const T*>(a.x) + lo;
  const uint8_t* const lb = kMask ? a.legal + lo : nullptr;

  u32x4 raw[kN];
  Word mk[kMask ? kN : 1];
  // Chunk t of a lane starts at (t * bd + tid) * kE.  Loads never branch: past
  // `last` (the last whole chunk's start) they repeat that chunk, and what lies
  // before a chunk's own start is dropped when it is used.
  int me = tid;  // (renewed for each pass)
  auto load = [&](int t, const T* x, const uint8_t* legal, int last) {
    // (an unsigned byte offset to a uniform base: no 64-bit address arithmetic)
    const uint32_t oc = min((t * bd + me) * kE, last);
    const uint32_t bytes = oc * static_cast<uint32_t>(sizeof(T));
    raw[t] = load_at<kStream, T, u32x4>(
        reinterpret_cast<const T*>(reinterpret_cast<const char*>(x) + bytes));
    if constexpr (kMask) mk[t] = *reinterpret_cast<const Word*>(legal + oc);
  };
  // The chunk's values, excluded ones -inf; true where it holds any.
  auto values = [&](int t, float (&x)[kE], int ln) {
    unpack<T>(raw[t], x);
    if constexpr (kMask) {
#pragma unroll
      for (int j = 0; j < kE; ++j)
        if (!mk[t].allows(j)) x[j] = neg_inf();
    }
    if ((t + 1) * bd * kE > ln) {
      const int o = (t * bd + me) * kE, oc = min(o, ln - kE);
#pragma unroll
      for (int j = 0; j < kE; ++j)
        if (oc + j < o) x[j] = neg_inf();
      if constexpr (kSums && kSecond && !kMask) raw[t] = pack<T, u32x4>(x);
    }
    if constexpr (kSums && kSecond && kMask) raw[t] = pack<T, u32x4>(x);
  };
  // The same again, once values() has left the exclusions in the registers.
  auto again = [&](int t, float (&x)[kE], int ln) {
    renew(raw[t]);
    if constexpr (kSums) unpack<T>(raw[t], x);
    else values(t, x, ln);
  };

  int64_t r = blockIdx.x;
  {
    const T* x = xb + r * a.ld;
    const uint8_t* legal = kMask ? lb + r * a.lld : nullptr;
#pragma unroll
    for (int t = 0; t < kN; ++t) load(t, x, legal, len - kE);
  }
  if constexpr (kTop) {
    if (tid < 64) top_lds.group[tid] = 0;
    __syncthreads();
  }

  RowValues<kOp> next = RowValues<kOp>::at(g, r);
  RawEntries<kTarget ? kHeld : 1> next_entries;
  if constexpr (kTarget) next_entries.load(g.t, r, tid, bd);

  for (int par = 0; r < a.n; r += gridDim.x, par ^= 1) {
    // The next row, loaded as this one's registers come free (after the last
    // row: one chunk, again and again).
    const bool more = r + gridDim.x < a.n;
    const int64_t rn = more ? r + gridDim.x : r;
    const T* const nx = xb + rn * a.ld;
    const uint8_t* const nl = kMask ? lb + rn * a.lld : nullptr;
    const int nlast = more ? len - kE : 0;

    const RowValues<kOp> val = next;
    next = RowValues<kOp>::at(g, rn);

    // -- listed entries, and their mass --
    int eid[kTarget ? kHeld : 1];
    float ez[kTarget ? kHeld : 1], ex[kTarget ? kHeld : 1];
    Mass mass{neg_inf(), 0.0f};
    float bad = 0.0f;
    Table tab{};
    if constexpr (kTarget) {
      const int k = g.t.k;
      next_entries.finish(g.t, tid, bd, a.v, eid, ez, bad);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) ex[i] = neg_inf();
      mass = mass_of(g.t, a.c, ez);
      for (int j = tid + kHeld * bd; j < k; j += bd) {
        const Entry e = target_entry(g.t, r, j);
        if (e.id >= a.v) bad = 1.0f;
        mass_add(g.t, a.c, e.z, mass);
      }
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (i * bd < k && eid[i] >= 0) ex[i] = logit<T>(a, r, eid[i]);
      // (ahead of the next row's chunks: loads come back in order)
      next_entries.load(g.t, rn, tid, bd);
      if constexpr (kGrad) {
        unsigned char* const base = dyn + static_cast<size_t>(par) * g.hash * 12;
        tab.key = reinterpret_cast<int32_t*>(base);
        tab.w = reinterpret_cast<float*>(base + static_cast<size_t>(g.hash) * 4);
        tab.x = reinterpret_cast<float*>(base + static_cast<size_t>(g.hash) * 8);
        tab.mask = g.hash - 1;
        table_clear(tab, tid, bd);
        if (tid == 0) twice[par] = 0;
      }
    }

    // -- the given action's logit --
    const int64_t given = val.given;
    float given_x = neg_inf();
    if constexpr (kEnt || kOp == kLogprobsGrad) {
      if (given >= 0 && given < a.v) given_x = logit<T>(a, r, given);
    }

    // -- the sums --
    // A lane's reference R is its largest x c so far, never below -kWild (what
    // is, adds nothing unless the whole row is: that one is wild, below).
    // Then d = x c - R is one operation an element and the sums are rescaled
    // once a chunk.
    Sums u{neg_inf(), 0.0f, 0.0f};
    float ref = -kWild;
    int best_o = 0;                       // start of the first chunk with the lane's maximum
    float chunk_max[kTop ? kN : 1];       // (NaN: see largest())
    if constexpr (kSums) {
      const int ln = renewed_scalar(len);
      renew(me);
#pragma unroll
      for (int t = 0; t < kN; ++t) {
        if constexpr (kTop) chunk_max[t] = neg_inf();
        if (t * bd * kE < ln) {
          float x[kE];
          values(t, x, ln);
          const float cm = largest<kE>(x);
          if constexpr (kTop) {  // (chunks past the row's end hold -inf)
            best_o = cm > u.m ? (t * bd + me) * kE : best_o;
            chunk_max[t] = cm;
          }
          u.m = fmaxf(u.m, cm);
          const float to = fmaxf(cm * a.c, ref);
          const float step = ref - to;
          const float f = exp2_(step);
          ref = to;
          float s = 0.0f, tc = 0.0f;
#pragma unroll
          for (int j = 0; j < kE; ++j) {
            const float d = fmaf(x[j], a.c, -to);
            const float e = exp2_(d);
            s += e;
            if constexpr (kEnt) tc = fmaf(e, kMask ? fmaxf(d, kFloor) : d, tc);
          }
          if constexpr (kEnt && !kMask) {
            // 0 * -inf: an excluded action (rare without a mask: not worth the
            // clamp on every element)
            if (__any(tc != tc)) {
              tc = 0.0f;
#pragma unroll
              for (int j = 0; j < kE; ++j) {
                const float d = fmaf(x[j], a.c, -to);
                tc = fmaf(exp2_(d), fmaxf(d, kFloor), tc);
              }
            }
          }
          if constexpr (kEnt) u.t = fmaf(f, fmaf(u.s, step, u.t), tc);
          u.s = fmaf(u.s, f, s);
        }
        if constexpr (!kSecond) load(t, nx, nl, nlast);
      }
    }

    // from R to the lane's exact m c (see mean_part())
    if constexpr (kSums) {
      if (ref > -kWild) {
        const float off = fmaf(u.m, a.c, -ref), e0 = exp2_(off), inv = __builtin_amdgcn_rcpf(e0);
        if constexpr (kEnt) u.t = inv * mean_part(u.s, u.t, e0, off);
        u.s = share(u.s, e0, inv);
      }
    }

    // -- across the lanes and waves --
    uint64_t lane_key = 0;
    if constexpr (kTop) {
      if (u.m > neg_inf()) lane_key = top_key(u.m, static_cast<uint32_t>(lo + best_o));
      if (nw > 1 && lane_key != 0)
        atomicMax(reinterpret_cast<unsigned long long*>(&top_lds.group[lane]),
                  static_cast<unsigned long long>(lane_key));
    }
    if constexpr (kSums) u = fold_sums<kEnt>(u, a.c);
    if constexpr (kTarget) {
      mass = mass_fold(g.t, a.c, mass, [](float z) { return fold64(z, Max{}); },
                       [](float z) { return fold64(z, Add{}); });
      bad = fold64(bad, Max{});
    }
    if (nw > 1) {
      if (lane == 0) {
        float* const q = red[par][wave];
        q[0] = u.m;
        q[1] = u.s;
        q[2] = u.t;
        q[3] = mass.z;
        q[4] = mass.s;
        q[5] = bad;
      }
      __syncthreads();
      const float* const q = red[par][lane & (kMaxWaves - 1)];
      const bool in = lane < nw;
      if constexpr (kSums) {
        u = in ? Sums{q[0], q[1], q[2]} : Sums{neg_inf(), 0.0f, 0.0f};
        u = fold_sums<kEnt>(u, a.c);
      }
      if constexpr (kTarget) {
        mass = in ? Mass{q[3], q[4]} : Mass{no_mass(g.t), 0.0f};
        mass = mass_fold(g.t, a.c, mass, [](float z) { return fold64(z, Max{}); },
                         [](float z) { return fold64(z, Add{}); });
        bad = fold64(in ? q[5] : 0.0f, Max{});
      }
    }
    float m, l;
    if constexpr (kSums) {
      // (well within -kWild: a lane below it has summed against that, not
      // against its own maximum, and must not count)
      if (u.m > neg_inf() && !(fabsf(u.m * a.c) <= kWild - 256.0f)) {
        // a wild row: once more, from memory
        u.s = u.t = 0.0f;
        for (int i = tid; i < len; i += bd) {
          const float d = (logit<T>(a, r, lo + i) - u.m) * a.c;
          const float e = exp2_(d);
          u.s += e;
          if constexpr (kEnt) u.t = fmaf(e, fmaxf(d, kFloor), u.t);
        }
        u.s = fold64(u.s, Add{});
        u.t = fold64(u.t, Add{});
        if (nw > 1) {
          __syncthreads();
          if (lane == 0) {
            red[par][wave][1] = u.s;
            red[par][wave][2] = u.t;
          }
          __syncthreads();
          u.s = u.t = 0.0f;
          for (int w = 0; w < nw; ++w) {
            u.s += red[par][w][1];
            u.t += red[par][w][2];
          }
        }
      }
      m = u.m == neg_inf() ? 0.0f : u.m;
      l = u.s == 0.0f ? 0.0f : log2f(u.s);
    } else {
      m = val.m;
      l = val.l;
    }

    // -- log probabilities --
    if constexpr (kOp == kLogprobs || kOp == kLogprobsTop) {
      const int64_t part = r * pt.parts + blockIdx.y;
      if (tid == 0) {
        if (g.sums != nullptr) {
          g.sums[part] = PartSums{u.m, u.s, u.t, 0.0f};
        } else {
          g.entropy[r] = kLn2 * (l - (u.s == 0.0f ? 0.0f : u.t / u.s));
          if (g.stats != nullptr) {
            g.stats[2 * r] = m;
            g.stats[2 * r + 1] = l;
          }
          if (g.actions != nullptr) {
            g.logprob[r] = given < 0 ? 0.0f
                           : given >= a.v ? __builtin_nanf("")
                                          : log_p(a, given_x, m, l);
          }
        }
      }
      if constexpr (kTop) {
        // The top-th largest of 64 lane maxima bounds the row's top-th largest
        // from below; ties are cut at the end of the chunk that holds it, so
        // what passes is a beginning of the order (value, then index) and has
        // `top` entries or all there are.  Usually a few more: they are ranked
        // by counting.  (The lanes' maxima are known from the sums; a selection
        // without the bound costs a pass over the row for each of `top`.)
        if (wave == 0) {
          const uint64_t key = nw == 1 ? lane_key : top_lds.group[lane];
          const float v = key == 0 ? neg_inf() : key_value(key);
          const int at = key == 0 ? 0x7FFFFFFF : static_cast<int>(key_index(key));
          const float tv = kth_bound(v, m, g.top);
          // of those at the bound, as many as `top` still needs, the first
          const uint64_t tied = __ballot(v == tv && key != 0);
          const int need = g.top - __builtin_popcountll(__ballot(v > tv));
          int cut = -kE;
          if (tied != 0 && need > 0) {
            const int mine = v == tv ? at : 0x7FFFFFFF;
            int rank = 0;
            if (tied & (tied - 1)) {
              for (int j = 0; j < 64; ++j) rank += __builtin_amdgcn_readlane(mine, j) < mine ? 1 : 0;
            }
            const uint64_t in = tied & __ballot(rank < need);
            // the last of them: the one with the largest start
            int far = (in >> lane & 1) != 0 ? mine : -1;
            for (int o = 32; o > 0; o >>= 1) far = max(far, __shfl_xor(far, o));
            cut = far;
          }
          top_lds.group[lane] = 0;
          if (lane == 0) {
            top_lds.bound = tv;
            top_lds.cut = cut + kE;
            top_lds.count = 0;
            top_lds.chunks = 0;
          }
        }
        __syncthreads();
        const bool odd = l != l;
        const float tv = top_lds.bound;
        const int ti = top_lds.cut - lo;
        const int ln = renewed_scalar(len);
        renew(me);
        // The chunks that hold them are few: listed, and read once more (their
        // registers have gone to the next row already), an element a lane.
#pragma unroll
        for (int t = 0; t < kN; ++t) {
          const float cm = chunk_max[t];
          const int o = (t * bd + me) * kE;
          if (!odd && (cm > tv || (cm == tv && o < ti && tv > neg_inf()))) {
            const uint32_t at = atomicAdd(&top_lds.chunks, 1u);
            if (at < kCandidates) top_lds.chunk[at] = o;
          }
        }
        __syncthreads();
        const int listed = static_cast<int>(top_lds.chunks);
        for (int i = tid; i < min(listed, kCandidates) * kE; i += bd) {
          const int o = top_lds.chunk[i / kE], e = min(o, ln - kE) + i % kE;
          const float x = logit<T>(a, r, lo + e);
          if (e >= o && (x > tv || (x == tv && e < ti))) {
            const uint32_t at = atomicAdd(&top_lds.count, 1u);
            if (at < kCandidates) top_lds.cand[at] = top_key(x, static_cast<uint32_t>(lo + e));
          }
        }
        __syncthreads();
        const int found = odd ? 0 : listed > kCandidates ? listed : static_cast<int>(top_lds.count);
        const auto put = [&](int rank, uint64_t key) {
          if (g.part_keys != nullptr) {
            g.part_keys[part * g.top + rank] = key;
            return;
          }
          g.top_action[r * g.top + rank] = key == 0 ? -1 : static_cast<int64_t>(key_index(key));
          g.top_logprob[r * g.top + rank] =
              odd ? l : key == 0 ? neg_inf() : log_p(a, key_value(key), m, l);
        };
        if (found <= kCandidates) {
          for (int i = tid; i < found; i += bd) {
            const uint64_t key = top_lds.cand[i];
            int rank = 0;
            for (int j = 0; j < found; ++j) rank += top_lds.cand[j] > key ? 1 : 0;
            if (rank < g.top) put(rank, key);
          }
          for (int i = found + tid; i < g.top; i += bd) put(i, 0);
        } else {
          // Hundreds of the largest values in fewer lanes than `top`: one
          // round over the row for each, from memory.
          uint64_t last = ~0ull;
          for (int k = 0; k < g.top; ++k) {
            uint64_t best = 0;
            for (int i = tid; i < len; i += bd) {
              const float x = logit<T>(a, r, lo + i);
              const uint64_t key = top_key(x, static_cast<uint32_t>(lo + i));
              if (x > neg_inf() && key < last && key > best) best = key;
            }
            best = fold64_max(best);
            __syncthreads();
            if (lane == 0) top_lds.cand[wave] = best;
            __syncthreads();
            for (int w = 0; w < nw; ++w) best = top_lds.cand[w] > best ? top_lds.cand[w] : best;
            if (tid == 0) put(k, best);
            last = best;
          }
        }
      }
    }

    // -- distillation: loss, and the listed weights --
    float f0 = 0.0f, f1 = 0.0f, scale = 0.0f, inv = 0.0f;
    if constexpr (kTarget) {
      inv = mass.s == 0.0f ? 0.0f : 1.0f / mass.s;
      if constexpr (kGrad) {
        scale = val.weight * a.inv_t;
        f0 = bad != 0.0f ? __builtin_nanf("") : scale * share(mass.s, mass.s, inv);
      }
    }
    // The entries' part in the loss, and their weights into the table (before the
    // gradient's pass, whose loads for the next row the logits' would wait for).
    [[maybe_unused]] const auto use_targets = [&](const auto& g) {
      float ce = 0.0f, h = 0.0f;
      const auto use = [&](int id, float z, float x) {
        const float q = share(target_mass(g.t, a.c, z, mass.z), mass.s, inv);
        if constexpr (kOp != kDistillGrad) {
          if (q != 0.0f) {
            if (id >= 0) ce -= q * log_p(a, x, m, l);
            h -= q * log_share(q);
          }
        }
        if constexpr (kGrad) {
          if (id >= lo && id < lo + len && x > neg_inf())
            if (!table_put(tab, id, -scale * q, x)) twice[par] = 1;
        }
      };
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (i * bd < g.t.k) use(eid[i], ez[i], ex[i]);
      for (int j = tid + kHeld * bd; j < g.t.k; j += bd) {
        const Entry e = target_entry(g.t, r, j);
        const int id = e.id < 0 || e.id >= a.v ? -1 : static_cast<int>(e.id);
        use(id, e.z, id < 0 ? neg_inf() : logit<T>(a, r, id));
      }
      if constexpr (kOp != kDistillGrad) {
        ce = fold64(ce, Add{});
        h = fold64(h, Add{});
        if (lane == 0) {
          red2[par][wave][0] = ce;
          red2[par][wave][1] = h;
        }
      }
    };
    [[maybe_unused]] const auto write_loss = [&](const auto& g) {  // after the barrier
      if (tid != 0) return;
      float ce = 0.0f, h = 0.0f;
      for (int w = 0; w < nw; ++w) {
        ce += red2[par][w][0];
        h += red2[par][w][1];
      }
      g.loss[r] = bad != 0.0f ? __builtin_nanf("") : ce;
      if (g.tent != nullptr) g.tent[r] = h;
      if (g.stats != nullptr) {
        g.stats[2 * r] = m;
        g.stats[2 * r + 1] = l;
      }
    };
    if constexpr (kTarget) use_targets(g);
    if constexpr (kOp == kDistill) {
      __syncthreads();
      write_loss(g);
    }

    // -- gradient of the log probabilities: factors and listed weights --
    int act = -1;
    float act_w = 0.0f, act_x = neg_inf();
    if constexpr (kOp == kLogprobsGrad) {
      float sum = 0.0f;
      if (g.gl != nullptr && given >= 0) {
        sum = given >= a.v ? __builtin_nanf("") : val.gl;
        if (given < a.v) {
          act = static_cast<int>(given);
          act_w = sum * a.inv_t;
          act_x = given_x;
        }
      }
      if (g.top > 0) {
        int64_t ti = -1;
        float gt = 0.0f;
        if (lane < g.top) {
          ti = g.top_action[r * g.top + lane];
          gt = ti >= 0 && ti < a.v ? g.gt[r * g.top + lane] : 0.0f;
        }
        sum += fold64(gt, Add{});
        unsigned char* const base = dyn + static_cast<size_t>(par) * 128 * 12;
        tab.key = reinterpret_cast<int32_t*>(base);
        tab.w = reinterpret_cast<float*>(base + 128 * 4);
        tab.x = reinterpret_cast<float*>(base + 128 * 8);
        tab.mask = 127;
        table_clear(tab, tid, bd);
        if (tid == 0) twice[par] = 0;
        __syncthreads();
        if (wave == 0 && ti >= lo && ti < lo + len) {
          const float x = logit<T>(a, r, ti);
          if (x > neg_inf() && !table_put(tab, static_cast<int>(ti), gt * a.inv_t, x)) twice[par] = 1;
        }
      }
      f0 = -(sum + (val.gh != 0.0f ? val.gh * val.entropy : 0.0f)) * a.inv_t;
      f1 = -val.gh * kLn2 * a.inv_t;
    }

    // -- the gradient --
    if constexpr (kGrad) {
      const Dense<false> dn{m, l, a.c, f0, f1};
      constexpr bool kLog = kOp == kLogprobsGrad;
      T* const gb = static_cast<T*>(g.grad) + r * g.grad_ld + lo;
      const int ln = renewed_scalar(len);
      renew(me);
#pragma unroll
      for (int t = 0; t < kN; ++t) {
        if (t * bd * kE < ln) {
          float x[kE], y[kE];
          again(t, x, ln);
          const int o = (t * bd + me) * kE, oc = min(o, ln - kE);
          if (dn.plain) {
#pragma unroll
            for (int j = 0; j < kE; ++j) y[j] = dn.template at<kLog>(x[j]);
          } else {
#pragma unroll
            for (int j = 0; j < kE; ++j) y[j] = dn.template any<kLog>(x[j]);
          }
          if (o + kE <= ln) {
            const uint32_t bytes = static_cast<uint32_t>(o) * static_cast<uint32_t>(sizeof(T));
            store_at<kStream>(reinterpret_cast<T*>(reinterpret_cast<char*>(gb) + bytes), pack<T, u32x4>(y));
          } else if (o < ln) {
#pragma unroll
            for (int j = 0; j < kE; ++j)
              if (oc + j >= o) gb[oc + j] = static_cast<T>(y[j]);
          }
        }
        load(t, nx, nl, nlast);
      }
      // the listed actions once more, with their weights (a barrier: after the
      // dense stores of whichever wave)
      const auto fix = [&](int id, float w, float x) {
        gb[id - lo] = static_cast<T>(dn.template any<kLog>(x) + w);
      };
      if constexpr (kTarget) {
        __syncthreads();
        if constexpr (kOp == kDistillFused) write_loss(g);
        if (twice[par] != 0) {
          // the entries in order, through the other row's table (at rest)
          unsigned char* const base = dyn + static_cast<size_t>(par ^ 1) * g.hash * 12;
          int32_t* const lid = reinterpret_cast<int32_t*>(base);
          float* const lw = reinterpret_cast<float*>(base + static_cast<size_t>(g.hash) * 4);
          float* const lx = reinterpret_cast<float*>(base + static_cast<size_t>(g.hash) * 8);
          table_clear(tab, tid, bd);
          for (int j = tid; j < g.t.k; j += bd) {
            const Entry e = target_entry(g.t, r, j);
            const bool in = e.id >= lo && e.id < lo + len;
            lid[j] = in ? static_cast<int32_t>(e.id) : -1;
            lx[j] = in ? logit<T>(a, r, e.id) : neg_inf();
            lw[j] = -scale * share(target_mass(g.t, a.c, e.z, mass.z), mass.s, inv);
          }
          __syncthreads();
          if (tid == 0)
            for (int j = 0; j < g.t.k; ++j)
              if (lid[j] >= 0 && lx[j] > neg_inf()) table_add(tab, lid[j], lw[j], lx[j]);
          __syncthreads();
        }
        for (int i = tid; i <= tab.mask; i += bd)
          if (tab.key[i] >= 0) fix(tab.key[i], tab.w[i], tab.x[i]);
      } else {
        __syncthreads();
        const bool mine = act >= lo && act < lo + len && act_x > neg_inf();
        if (g.top == 0) {
          if (tid == 0 && mine) fix(act, act_w, act_x);
        } else {
          const bool again_ = twice[par] != 0;
          if (again_) {
            __syncthreads();
            table_clear(tab, tid, bd);
            __syncthreads();
          }
          if (tid == 0) {
            if (again_)
              for (int j = 0; j < g.top; ++j) {
                const int64_t id = g.top_action[r * g.top + j];
                if (id < lo || id >= lo + len) continue;
                const float x = logit<T>(a, r, id);
                if (x > neg_inf())
                  table_add(tab, static_cast<int>(id), g.gt[r * g.top + j] * a.inv_t, x);
              }
            if (mine) table_add(tab, act, act_w, act_x);
          }
          __syncthreads();
          for (int i = tid; i <= tab.mask; i += bd)
            if (tab.key[i] >= 0) fix(tab.key[i], tab.w[i], tab.x[i]);
        }
      }
    }
  }
}

// ---- rows of up to kWaveMax actions: a wave each ----

// kC chunks of 8 or 16 bytes (W) a lane, the values in registers as floats; the
// next row's chunks are under way while a row is worked on.  No barrier is
// needed: what goes through LDS stays within the wave, whose accesses are in
// order (fence() keeps the compiler to it).  The vector units are what a row
// waits for here: 366 instructions a row of 12 actions a lane with the mask and
// the top actions, a third of them the elements' own, the rest the row's folds,
// bound, ranking and addresses (65536 x 768 masked bf16, top 8: 52 us, units three
// quarters busy; 32 us is the memory's share), so rows take the smallest kernel
// that holds them and only the last chunk is ever short, of six and eight the last
// two (the same in two chunks of 16 bytes rather than three of 8: 4 us more).
// Against a workgroup of k_rows it saves the barriers: 44739 x 1500 f32, top 8: 99
// -> 54 us, loss and gradient: 152 -> 115 us.
// Waves a SIMD that the registers must leave room for (left alone, the compiler
// keeps every address it could compute again): what the dependent steps of a row
// leave idle, other rows fill (8 rather than 7 at that size: 57 -> 53 us).
template <bool kMask, int kX, int kOp>
constexpr int kWaveRoom = kOp == kLogprobs || kOp == kLogprobsTop ? (kX <= 12 ? 8 : kX <= 16 ? 6 : 4)
                          : kOp == kDistill                       ? (kX <= 8 ? 6 : kX <= 16 ? 5 : 4)
                          : kX <= 8                               ? (kMask ? 4 : 5)
                          : kX <= 16                              ? 4
                                                                  : 2;
template <class T, class W, int kC>
constexpr int kWaveEach = kC * static_cast<int>(sizeof(W) / sizeof(T));  // elements a lane
template <class T, bool kMask, class W, int kC, int kOp>
__global__ __launch_bounds__(64, (kWaveRoom<kMask, kWaveEach<T, W, kC>, kOp>)) void k_wave(
    Rows a, ArgsOf<kOp> g) {
  constexpr int kE = static_cast<int>(sizeof(W) / sizeof(T)), kX = kC * kE;
  constexpr bool kSums = kOp != kLogprobsGrad && kOp != kDistillGrad;
  constexpr bool kGrad = kOp == kLogprobsGrad || kOp == kDistillGrad || kOp == kDistillFused;
  constexpr bool kLp = kOp == kLogprobs || kOp == kLogprobsTop;
  constexpr bool kTarget = kOp == kDistill || kOp == kDistillFused || kOp == kDistillGrad;
  constexpr int kHeld = 6;  // target entries a lane keeps in registers
  using Word = MaskWord<kE>;
  // The row's values, then its listed weights: chunk (t, lane) at
  // (t * 64 + lane) * kE, the row's last actions where their chunk has them.
  __shared__ __attribute__((aligned(16))) float row[kTarget || kGrad ? 64 * kX : 1];
  __shared__ Found cand[kOp == kLogprobsTop ? kWaveCandidates + 64 : 1];
  __shared__ uint64_t keys[kOp == kLogprobsTop ? kWaveCandidates : 1];
  const int lane = threadIdx.x;
  const int last = a.v - kE;
  const auto fence = [] { __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront"); };

  W raw[kC];
  Word mk[kMask ? kC : 1];
  const auto load = [&](int64_t r) {
    const T* const x = static_cast<const T*>(a.x) + r * a.ld;
    const uint8_t* const legal = kMask ? a.legal + r * a.lld : nullptr;
#pragma unroll
    for (int t = 0; t < kC; ++t) {
      const int oc = min((t * 64 + lane) * kE, last);
      raw[t] = load_at<false, T, W>(x + oc);
      if constexpr (kMask) mk[t] = *reinterpret_cast<const Word*>(legal + oc);
    }
  };
  // Where an action is in `row`: the last, shifted chunk holds those from
  // `edge` on.
  const int edge = a.v / kE * kE, shift = (kE - a.v % kE) % kE;
  const auto slot = [&](int id) { return id + (id >= edge ? shift : 0); };

  // Chunks that every row of this kernel fills (a smaller kernel takes the rest),
  // and how many elements of the others come before their own start (see load()).
  constexpr int kFull = kC - (kC > 4 ? 2 : 1);
  int drop[kC - kFull];
#pragma unroll
  for (int t = kFull; t < kC; ++t)
    drop[t - kFull] = (t * 64 + lane) * kE - min((t * 64 + lane) * kE, last);

  RowValues<kOp> next = RowValues<kOp>::at(g, blockIdx.x);
  load(blockIdx.x);
  for (int64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    // -- the row's values --
    int me = lane;  // (renewed: offsets are cheaper computed than kept)
    renew(me);
    float x[kX];
#pragma unroll
    for (int t = 0; t < kC; ++t) {
      float v[kE];
      unpack<T>(raw[t], v);
#pragma unroll
      for (int j = 0; j < kE; ++j) x[t * kE + j] = v[j];
      if constexpr (kMask) {
#pragma unroll
        for (int j = 0; j < kE; ++j)
          if (!mk[t].allows(j)) x[t * kE + j] = neg_inf();
      }
      if (t >= kFull) {
#pragma unroll
        for (int j = 0; j < kE; ++j)
          if (j < drop[t - kFull]) x[t * kE + j] = neg_inf();
      }
    }
    // -- what else the row needs from memory, issued ahead of the next row's loads
    // (the given action's logit is waited for at its mask byte, which logit()
    // branches on; the target's entries where they are used) --
    const RowValues<kOp> val = next;
    const int64_t given = val.given;
    float given_x = neg_inf();
    if constexpr (kLp || kOp == kLogprobsGrad) {
      if (given >= 0 && given < a.v) given_x = logit<T>(a, r, given);
    }
    int eid[kTarget ? kHeld : 1];
    float ez[kTarget ? kHeld : 1];
    Mass mass{neg_inf(), 0.0f};
    float bad = 0.0f;
    const auto entry_id = [&](const Entry& e) {
      return e.id < 0 || e.id >= a.v ? -1 : static_cast<int>(e.id);
    };
    if constexpr (kTarget) {
      target_entries<kHeld>(g.t, r, lane, 64, a.v, eid, ez, bad);
    }
    if (r + gridDim.x < a.n) {
      next = RowValues<kOp>::at(g, r + gridDim.x);
      load(r + gridDim.x);
    }

    // -- the sums --
    float m, l, mean = 0.0f, lane_max = neg_inf();
    if constexpr (kSums) {
#pragma unroll
      for (int i = 0; i < kX; ++i) lane_max = fmaxf(lane_max, x[i]);
      m = fold64(lane_max, Max{});
      if (m == neg_inf()) m = 0.0f;  // empty, or only NaN
      float s = 0.0f, u = 0.0f, off = 0.0f, e0 = 1.0f;
      const float ref = m * a.c;
      if (fabsf(ref) <= kWild) {
        off = fmaf(m, a.c, -ref);
        e0 = exp2_(off);
#pragma unroll
        for (int i = 0; i < kX; ++i) {
          const float d = fmaf(x[i], a.c, -ref);
          const float e = exp2_(d);
          s += e;
          if constexpr (kLp) u = fmaf(e, fmaxf(d, kFloor), u);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kX; ++i) {
          const float d = (x[i] - m) * a.c;
          const float e = exp2_(d);
          s += e;
          if constexpr (kLp) u = fmaf(e, fmaxf(d, kFloor), u);
        }
      }
      s = fold64(s, Add{});
      l = s == 0.0f ? 0.0f : log2f(share(s, e0, __builtin_amdgcn_rcpf(e0)));
      if constexpr (kLp) mean = s == 0.0f ? 0.0f : mean_part(s, fold64(u, Add{}), e0, off) / s;
    } else {
      m = val.m;
      l = val.l;
    }

    if constexpr (kLp) {
      if (lane == 0) {
        g.entropy[r] = kLn2 * (l - mean);
        if (g.stats != nullptr) {
          g.stats[2 * r] = m;
          g.stats[2 * r + 1] = l;
        }
        if (g.actions != nullptr)
          g.logprob[r] = given < 0 ? 0.0f
                         : given >= a.v ? __builtin_nanf("")
                                        : log_p(a, given_x, m, l);
      }
    }
    if constexpr (kOp == kLogprobsTop) {
      // Everything from a lower bound of the top-th largest value on, listed
      // (usually a few more than `top`) and ranked by counting.
      const bool odd = l != l;
      const auto put = [&](int rank, uint64_t key) {
        g.top_action[r * g.top + rank] = key == 0 ? -1 : static_cast<int64_t>(key_index(key));
        g.top_logprob[r * g.top + rank] =
            odd ? l : key == 0 ? neg_inf() : log_p(a, key_value(key), m, l);
      };
      const float bound = fmaxf(kth_bound(lane_max, m, g.top), kLowest);
      int found = 0;
      renew(me);
      if (!odd) {
#pragma unroll
        for (int t = 0; t < kC; ++t) {
          const int oc = min((t * 64 + me) * kE, last);
#pragma unroll
          for (int j = 0; j < kE; ++j) {
            const bool in = x[t * kE + j] >= bound;
            const uint64_t hit = __ballot(in);
            if (hit != 0) {
              const int at = __builtin_amdgcn_mbcnt_hi(
                  static_cast<uint32_t>(hit >> 32),
                  __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(hit), found));
              if (in && found <= kWaveCandidates) cand[at] = Found{x[t * kE + j], oc + j};
              found += __builtin_popcountll(hit);
            }
          }
        }
      }
      if (found <= kWaveCandidates) {
        fence();
        const int whole = (found + 63) & ~63;
        for (int i = lane; i < whole; i += 64) {
          const Found f = cand[i];  // (past `found`: not used)
          keys[i] = i < found ? top_key(f.x, static_cast<uint32_t>(f.i)) : 0;
        }
        fence();
        for (int i = lane; i < whole; i += 64) {
          const uint64_t key = keys[i];
          int rank = 0;
          for (int j = 0; j < found; j += 8) {
#pragma unroll
            for (int q = 0; q < 8; ++q) rank += keys[j + q] > key ? 1 : 0;
          }
          if (i < found && rank < g.top) put(rank, key);
        }
        if (lane >= found && lane < g.top) put(lane, 0);
        fence();
      } else {
        // Equal values at the bound: one round over the registers for each.
        uint64_t prev = ~0ull;
        for (int k = 0; k < g.top; ++k) {
          uint64_t best = 0;
          renew(me);
#pragma unroll
          for (int i = 0; i < kX; ++i) {
            renew(x[i]);
            const int o = (i / kE * 64 + me) * kE;
            const uint64_t key = top_key(x[i], static_cast<uint32_t>(min(o, last) + i % kE));
            if (x[i] > neg_inf() && key < prev && key > best) best = key;
          }
          best = fold64_max(best);
          if (lane == 0) put(k, best);
          prev = best;
        }
      }
    }

    // -- the listed entries --
    float f0 = 0.0f, f1 = 0.0f;
    const auto clear = [&] {
#pragma unroll
      for (int t = 0; t < kX / 2; ++t)
        *reinterpret_cast<u32x2*>(row + (t * 64 + lane) * 2) = u32x2{0, 0};
    };
    [[maybe_unused]] int* const tag = reinterpret_cast<int*>(row);
    if constexpr (kTarget) {
      const int k = g.t.k;
      // f(id, z, number, i) for each of this lane's entries
      const auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
          if (i * 64 < k) f(eid[i], ez[i], lane + i * 64);
        for (int j = lane + kHeld * 64; j < k; j += 64) {
          const Entry e = target_entry(g.t, r, j);
          f(entry_id(e), e.z, j);
        }
      };
      for (int j = lane + kHeld * 64; j < k; j += 64)
        if (target_entry(g.t, r, j).id >= a.v) bad = 1.0f;
      bool clash = false;
      mass = mass_of(g.t, a.c, ez);
      for (int j = lane + kHeld * 64; j < k; j += 64)
        mass_add(g.t, a.c, target_entry(g.t, r, j).z, mass);
      each([&](int id, float z, int j) {
        if (kGrad && g.t.ids != nullptr && id >= 0) tag[slot(id)] = j;
      });
      if constexpr (kGrad) {
        // an entry that finds another's number shares its action
        if (g.t.ids != nullptr) {
          fence();
          int c = 0;
          each([&](int id, float z, int j) {
            if (id >= 0) c |= tag[slot(id)] != j;
          });
          clash = __ballot(c) != 0;
          fence();
        }
      }
#pragma unroll
      for (int t = 0; t < kC; ++t)
#pragma unroll
        for (int j = 0; j < kE; ++j) row[(t * 64 + lane) * kE + j] = x[t * kE + j];
      fence();
      mass = mass_fold(g.t, a.c, mass, [](float z) { return fold64(z, Max{}); },
                       [](float z) { return fold64(z, Add{}); });
      bad = fold64(bad, Max{});
      const float inv = mass.s == 0.0f ? 0.0f : 1.0f / mass.s;
      float scale = 0.0f, ce = 0.0f, h = 0.0f;
      if constexpr (kGrad) {
        scale = val.weight * a.inv_t;
        f0 = bad != 0.0f ? __builtin_nanf("") : scale * share(mass.s, mass.s, inv);
      }
      float ew[kGrad ? kHeld : 1];  // the weights, until the values are read
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        if (i * 64 < k) {
          const float q = share(target_mass(g.t, a.c, ez[i], mass.z), mass.s, inv);
          const float xi = eid[i] >= 0 ? row[slot(eid[i])] : neg_inf();
          if constexpr (kOp != kDistillGrad) {
            if (q != 0.0f) {
              if (eid[i] >= 0) ce -= q * log_p(a, xi, m, l);
              h -= q * log_share(q);
            }
          }
          if constexpr (kGrad) {
            ew[i] = -scale * q;
            if (!(xi > neg_inf())) eid[i] = -1;
          }
        }
      }
      for (int j = lane + kHeld * 64; j < k; j += 64) {
        const Entry e = target_entry(g.t, r, j);
        const int id = entry_id(e);
        const float q = share(target_mass(g.t, a.c, e.z, mass.z), mass.s, inv);
        if constexpr (kOp != kDistillGrad) {
          if (q != 0.0f) {
            if (id >= 0) ce -= q * log_p(a, row[slot(id)], m, l);
            h -= q * log_share(q);
          }
        }
      }
      if constexpr (kOp != kDistillGrad) {
        ce = fold64(ce, Add{});
        h = fold64(h, Add{});
        if (lane == 0) {
          g.loss[r] = bad != 0.0f ? __builtin_nanf("") : ce;
          if (g.tent != nullptr) g.tent[r] = h;
          if (g.stats != nullptr) {
            g.stats[2 * r] = m;
            g.stats[2 * r + 1] = l;
          }
        }
      }
      fence();
      if constexpr (kGrad) {
        clear();
        fence();
        if (!clash) {
#pragma unroll
          for (int i = 0; i < kHeld; ++i)
            if (i * 64 < k && eid[i] >= 0) row[slot(eid[i])] = ew[i];
          for (int j = lane + kHeld * 64; j < k; j += 64) {
            const Entry e = target_entry(g.t, r, j);
            const int id = entry_id(e);
            if (id >= 0 && logit<T>(a, r, id) > neg_inf())
              row[slot(id)] = -scale * share(target_mass(g.t, a.c, e.z, mass.z), mass.s, inv);
          }
        } else {  // in list order
#pragma unroll
          for (int i = 0; i < kHeld; ++i) {
            for (int q = 0; q < 64 && q + i * 64 < k; ++q) {
              const int id = __builtin_amdgcn_readlane(eid[i], q);
              const float w = lane_at(ew[i], q);
              if (id >= 0 && lane == 0) row[slot(id)] += w;
            }
          }
          for (int j = kHeld * 64; j < k && lane == 0; ++j) {
            const Entry e = target_entry(g.t, r, j);
            const int id = entry_id(e);
            if (id >= 0 && logit<T>(a, r, id) > neg_inf())
              row[slot(id)] -= scale * share(target_mass(g.t, a.c, e.z, mass.z), mass.s, inv);
          }
        }
        fence();
      }
    }
    if constexpr (kOp == kLogprobsGrad) {
      const bool in = g.gl != nullptr && given >= 0 && given < a.v;
      const float gl = in ? val.gl : 0.0f;
      float sum = g.gl != nullptr && given >= a.v ? __builtin_nanf("") : gl;
      clear();
      fence();
      if (g.top > 0) {
        int64_t ti = -1;
        float gt = 0.0f;
        if (lane < g.top) {
          ti = g.top_action[r * g.top + lane];
          if (ti >= a.v) ti = -1;
          if (ti >= 0) gt = g.gt[r * g.top + lane];
        }
        sum += fold64(gt, Add{});
        if (ti >= 0) tag[slot(static_cast<int>(ti))] = lane;
        fence();
        const bool clash = __ballot(ti >= 0 && tag[slot(static_cast<int>(ti))] != lane) != 0;
        fence();
        const bool on = ti >= 0 && logit<T>(a, r, ti) > neg_inf();
        if (ti >= 0) row[slot(static_cast<int>(ti))] = clash || !on ? 0.0f : gt * a.inv_t;
        fence();
        if (clash && lane == 0)
          for (int j = 0; j < g.top; ++j) {
            const int64_t id = g.top_action[r * g.top + j];
            if (id >= 0 && id < a.v && logit<T>(a, r, id) > neg_inf())
              row[slot(static_cast<int>(id))] += g.gt[r * g.top + j] * a.inv_t;
          }
        fence();
      }
      if (lane == 0 && in && given_x > neg_inf()) row[slot(static_cast<int>(given))] += gl * a.inv_t;
      fence();
      f0 = -(sum + (val.gh != 0.0f ? val.gh * val.entropy : 0.0f)) * a.inv_t;
      f1 = -val.gh * kLn2 * a.inv_t;
    }

    // -- the gradient --
    if constexpr (kGrad) {
      constexpr bool kLog = kOp == kLogprobsGrad;
      const Dense<false> dn{m, l, a.c, f0, f1};
      T* const gb = static_cast<T*>(g.grad) + r * g.grad_ld;
      renew(me);
#pragma unroll
      for (int t = 0; t < kC; ++t) {
        float y[kE];
#pragma unroll
        for (int j = 0; j < kE; ++j) y[j] = row[(t * 64 + me) * kE + j];
        if (dn.plain) {
#pragma unroll
          for (int j = 0; j < kE; ++j) y[j] += dn.template at<kLog>(x[t * kE + j]);
        } else {
#pragma unroll
          for (int j = 0; j < kE; ++j) y[j] += dn.template any<kLog>(x[t * kE + j]);
        }
        const int o = (t * 64 + me) * kE;
        if (t < kFull || o + kE <= a.v) {
          store_at<false>(gb + o, pack<T, W>(y));
        } else if (o < a.v) {
#pragma unroll
          for (int j = 0; j < kE; ++j)
            if (last + j >= o) gb[last + j] = static_cast<T>(y[j]);
        }
      }
      fence();
    }
  }
}

// ---- joining a row's parts ----

// One workgroup of kJoin lanes a row: the parts' sums (a lane each), then their
// top lists or the loss.  All latency: 5 us for one row of 16 parts and its top
// 20, 7 us for 512 rows of 7 parts and 256 targets.
constexpr int kJoin = 256;
constexpr int kJoinGridX = 1 << 20;

template <class T, bool kLoss>
__global__ __launch_bounds__(kJoin) void k_join(Rows a, JoinArgs g) {
  __shared__ uint64_t cand[kLoss ? 1 : kMaxSplit * OS_AZ_MAX_TOP];
  __shared__ uint32_t count;
  __shared__ float red[kJoin / 64][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // (a grid of more than 2^32 lanes along x is not launched)
  const int64_t r = blockIdx.y * int64_t{kJoinGridX} + blockIdx.x;
  if (r >= a.n) return;
  const PartSums* const ps = g.lp.sums + r * g.parts;
  Sums u{neg_inf(), 0.0f, 0.0f};
  if (lane < g.parts) u = Sums{ps[lane].m, ps[lane].s, ps[lane].t};
  u = fold_sums<!kLoss>(u, a.c);
  const float m = u.m == neg_inf() ? 0.0f : u.m;
  const float l = u.s == 0.0f ? 0.0f : log2f(u.s);
  float* const stats = kLoss ? g.ds.stats : g.lp.stats;
  if (tid == 0 && stats != nullptr) {
    stats[2 * r] = m;
    stats[2 * r + 1] = l;
  }
  if constexpr (!kLoss) {
    const LogprobArgs& q = g.lp;
    if (tid == 0) {
      q.entropy[r] = kLn2 * (l - (u.s == 0.0f ? 0.0f : u.t / u.s));
      if (q.actions != nullptr) {
        const int64_t id = get_id(q.actions, q.wide, r);
        q.logprob[r] = id < 0 ? 0.0f
                       : id >= a.v ? __builtin_nanf("")
                                   : log_p(a, logit<T>(a, r, id), m, l);
      }
      count = 0;
    }
    if (q.top == 0) return;
    // Each list is in order.  With `deep` = ceil(top / parts) entries a list,
    // the ceil(top / deep)-th largest of the lists' deep-th entries has at
    // least `top` entries at or above it.
    const int deep = (q.top + g.parts - 1) / g.parts;
    const int need = (q.top + deep - 1) / deep;
    const uint64_t* const keys = q.part_keys + r * g.parts * q.top;
    const uint64_t lim = kth64(lane < g.parts ? keys[lane * q.top + deep - 1] : 0, need);
    __syncthreads();
    const bool odd = l != l;
    if (!odd)
      for (int i = tid; i < g.parts * q.top; i += kJoin) {
        const uint64_t k = keys[i];
        if (k != 0 && k >= lim) cand[atomicAdd(&count, 1u)] = k;
      }
    __syncthreads();
    const int found = static_cast<int>(count);
    const auto put = [&](int rank, uint64_t key) {
      q.top_action[r * q.top + rank] = key == 0 ? -1 : static_cast<int64_t>(key_index(key));
      q.top_logprob[r * q.top + rank] =
          odd ? l : key == 0 ? neg_inf() : log_p(a, key_value(key), m, l);
    };
    for (int i = tid; i < found; i += kJoin) {
      const uint64_t key = cand[i];
      int rank = 0;
      for (int j = 0; j < found; ++j) rank += cand[j] > key ? 1 : 0;
      if (rank < q.top) put(rank, key);
    }
    for (int i = found + tid; i < q.top; i += kJoin) put(i, 0);
  } else {
    const DistillArgs& q = g.ds;
    Mass mass{no_mass(q.t), 0.0f};
    float bad = 0.0f;
    for (int j = tid; j < q.t.k; j += kJoin) {
      const Entry e = target_entry(q.t, r, j);
      if (e.id >= a.v) bad = 1.0f;
      mass_add(q.t, a.c, e.z, mass);
    }
    const auto maxf = [](float z) { return fold64(z, Max{}); };
    const auto addf = [](float z) { return fold64(z, Add{}); };
    mass = mass_fold(q.t, a.c, mass, maxf, addf);
    bad = fold64(bad, Max{});
    if (lane == 0) {
      red[wave][0] = mass.z;
      red[wave][1] = mass.s;
      red[wave][2] = bad;
    }
    __syncthreads();
    const bool in = lane < kJoin / 64;
    const float* const w0 = red[lane & (kJoin / 64 - 1)];
    mass = in ? Mass{w0[0], w0[1]} : Mass{no_mass(q.t), 0.0f};
    bad = fold64(in ? w0[2] : 0.0f, Max{});
    mass = mass_fold(q.t, a.c, mass, maxf, addf);
    const float inv = mass.s == 0.0f ? 0.0f : 1.0f / mass.s;
    float ce = 0.0f, h = 0.0f;
    for (int j = tid; j < q.t.k; j += kJoin) {
      const Entry e = target_entry(q.t, r, j);
      const float p = share(target_mass(q.t, a.c, e.z, mass.z), mass.s, inv);
      if (p == 0.0f) continue;
      if (e.id >= 0 && e.id < a.v) ce -= p * log_p(a, logit<T>(a, r, e.id), m, l);
      h -= p * log_share(p);
    }
    ce = fold64(ce, Add{});
    h = fold64(h, Add{});
    __syncthreads();
    if (lane == 0) {
      red[wave][0] = ce;
      red[wave][1] = h;
    }
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kJoin / 64; ++w) {
        ce += red[w][0];
        h += red[w][1];
      }
      q.loss[r] = bad != 0.0f ? __builtin_nanf("") : ce;
      if (q.tent != nullptr) q.tent[r] = h;
    }
  }
}

// ---- rows of up to kTinyMax actions ----

// 16 lanes a row (one DPP row: reductions need no LDS), four elements a lane,
// 16 apart; 16 rows a workgroup.  A wave a row would leave most lanes idle at
// these sizes, a lane a row would leave the card empty at a few thousand rows
// (16384 x 7 masked f32, top 3: 4.7 us, most of it a launch's own).
constexpr int kTinyBlock = 256;
constexpr int kTinyRows = kTinyBlock / 16;

template <class T, int kOp>
__global__ __launch_bounds__(kTinyBlock) void k_tiny(Rows a, ArgsOf<kOp> g) {
  constexpr bool kSums = kOp != kLogprobsGrad && kOp != kDistillGrad;
  constexpr bool kGrad = kOp == kLogprobsGrad || kOp == kDistillGrad || kOp == kDistillFused;
  constexpr bool kTarget = kOp == kDistill || kOp == kDistillFused || kOp == kDistillGrad;
  constexpr int kEach = kTinyMax / 16;
  __shared__ float lds[kGrad ? kTinyRows : 1][kTinyMax];
  const int tid = threadIdx.x, l16 = tid & 15, sub = tid >> 4;
  float* const dq = lds[kGrad ? sub : 0];
  const Max maxf{};
  const Add addf{};
  // Whole workgroups go round together (barriers): a row past the end repeats
  // the last one and writes nothing.
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * kTinyRows; r0 < a.n;
       r0 += static_cast<int64_t>(gridDim.x) * kTinyRows) {
    const bool live = r0 + sub < a.n;
    const int64_t r = live ? r0 + sub : a.n - 1;
    float x[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      x[e] = neg_inf();
      const int i = l16 + 16 * e;
      if (16 * e < a.v && i < a.v) x[e] = logit<T>(a, r, i);
    }
    float m, l, mean = 0.0f;
    if constexpr (kSums) {
      float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      mx = fold16(mx, maxf);
      m = mx == neg_inf() ? 0.0f : mx;  // empty, or only NaN
      float s = 0.0f, t = 0.0f;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const float d = (x[e] - m) * a.c;
        const float p = exp2_(d);
        s += p;
        t = fmaf(p, fmaxf(d, kFloor), t);
      }
      s = fold16(s, addf);
      t = fold16(t, addf);
      l = s == 0.0f ? 0.0f : log2f(s);
      mean = s == 0.0f ? 0.0f : t / s;
    } else {
      m = g.stats[2 * r];
      l = g.stats[2 * r + 1];
    }
    if constexpr (kOp == kLogprobs || kOp == kLogprobsTop) {
      if (l16 == 0 && live) {
        g.entropy[r] = kLn2 * (l - mean);
        if (g.stats != nullptr) {
          g.stats[2 * r] = m;
          g.stats[2 * r + 1] = l;
        }
        if (g.actions != nullptr) {
          const int64_t id = get_id(g.actions, g.wide, r);
          g.logprob[r] = id < 0 ? 0.0f
                         : id >= a.v ? __builtin_nanf("")
                                     : log_p(a, logit<T>(a, r, id), m, l);
        }
      }
      if constexpr (kOp == kLogprobsTop) {
        const bool odd = l != l;
        for (int k = 0; k < g.top; ++k) {
          float best = odd ? neg_inf() : fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          best = fold16(best, maxf);
          uint32_t at = 0xFFFFFFFFu;
#pragma unroll
          for (int e = kEach - 1; e >= 0; --e)
            if (x[e] == best && best > neg_inf()) at = static_cast<uint32_t>(l16 + 16 * e);
          at = fold16(at, MinU{});
#pragma unroll
          for (int e = 0; e < kEach; ++e)
            if (static_cast<uint32_t>(l16 + 16 * e) == at) x[e] = neg_inf();
          if (l16 == 0 && live) {
            const bool none = best == neg_inf();
            g.top_action[r * g.top + k] = none ? -1 : static_cast<int64_t>(at);
            g.top_logprob[r * g.top + k] = odd ? l : none ? best : log_p(a, best, m, l);
          }
        }
      }
    }
    float f0 = 0.0f, f1 = 0.0f;
    if constexpr (kGrad) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) dq[l16 + 16 * e] = 0.0f;
      __syncthreads();
    }
    if constexpr (kTarget) {
      Mass mass{no_mass(g.t), 0.0f};
      float bad = 0.0f;
      int* const tag = reinterpret_cast<int*>(dq);
      for (int j = l16; j < g.t.k; j += 16) {
        const Entry e = target_entry(g.t, r, j);
        if (e.id >= a.v) bad = 1.0f;
        else if (kGrad && e.id >= 0) tag[e.id] = j;
        mass_add(g.t, a.c, e.z, mass);
      }
      mass = mass_fold(g.t, a.c, mass, [&](float z) { return fold16(z, maxf); },
                       [&](float z) { return fold16(z, addf); });
      bad = fold16(bad, maxf);
      const float inv = mass.s == 0.0f ? 0.0f : 1.0f / mass.s;
      float scale = 0.0f;
      if constexpr (kGrad)
        scale = (g.weight != nullptr ? g.weight[r * g.weight_stride] : 1.0f) * a.inv_t;
      float clash = 0.0f;
      if constexpr (kGrad) {
        // an entry that finds another's number shares its action
        __syncthreads();
        for (int j = l16; j < g.t.k; j += 16) {
          const int64_t id = g.t.ids != nullptr ? get_id(g.t.ids, g.t.wide, r * g.t.ids_ld + j) : j;
          if (id >= 0 && id < a.v && tag[id] != j) clash = 1.0f;
        }
        clash = fold16(clash, maxf);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e) dq[l16 + 16 * e] = 0.0f;
        __syncthreads();
      }
      float ce = 0.0f, h = 0.0f;
      for (int j = l16; j < g.t.k; j += 16) {
        const Entry e = target_entry(g.t, r, j);
        const float q = share(target_mass(g.t, a.c, e.z, mass.z), mass.s, inv);
        const bool in = e.id >= 0 && e.id < a.v;
        if constexpr (kOp != kDistillGrad) {
          if (q != 0.0f) {
            if (in) ce -= q * log_p(a, logit<T>(a, r, e.id), m, l);
            h -= q * log_share(q);
          }
        }
        if (kGrad && in && clash == 0.0f) dq[e.id] = -scale * q;
      }
      if constexpr (kOp != kDistillGrad) {
        ce = fold16(ce, addf);
        h = fold16(h, addf);
        if (l16 == 0 && live) {
          g.loss[r] = bad != 0.0f ? __builtin_nanf("") : ce;
          if (g.tent != nullptr) g.tent[r] = h;
          if (g.stats != nullptr) {
            g.stats[2 * r] = m;
            g.stats[2 * r + 1] = l;
          }
        }
      }
      if constexpr (kGrad) {
        if (clash != 0.0f && l16 == 0)
          for (int j = 0; j < g.t.k; ++j) {
            const Entry e = target_entry(g.t, r, j);
            if (e.id >= 0 && e.id < a.v)
              dq[e.id] -= scale * share(target_mass(g.t, a.c, e.z, mass.z), mass.s, inv);
          }
        f0 = bad != 0.0f ? __builtin_nanf("") : scale * share(mass.s, mass.s, inv);
        __syncthreads();
      }
    }
    if constexpr (kOp == kLogprobsGrad) {
      const int64_t id = g.actions != nullptr && g.gl != nullptr ? get_id(g.actions, g.wide, r) : -1;
      float sum = id >= a.v ? __builtin_nanf("") : 0.0f;
      const float gl = id >= 0 && id < a.v ? g.gl[r * g.gls] : 0.0f;
      sum += gl;
      if (l16 == 0) {  // (in list order: an action may be met twice)
        for (int j = 0; j < g.top; ++j) {
          const int64_t ti = g.top_action[r * g.top + j];
          if (ti < 0 || ti >= a.v) continue;
          const float w = g.gt[r * g.top + j];
          sum += w;
          dq[ti] += w * a.inv_t;
        }
        if (id >= 0 && id < a.v) dq[id] += gl * a.inv_t;
      }
      sum = __shfl(sum, tid & 48);  // the row's first lane's
      const float gh = g.gh != nullptr ? g.gh[r * g.ghs] : 0.0f;
      f0 = -(sum + (gh != 0.0f ? gh * g.entropy[r] : 0.0f)) * a.inv_t;
      f1 = -gh * kLn2 * a.inv_t;
      __syncthreads();
    }
    if constexpr (kGrad) {
      const Dense<true> dn{m, l, a.c, f0, f1};
      T* const gb = static_cast<T*>(g.grad) + r * g.grad_ld;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int i = l16 + 16 * e;
        if (i < a.v && live) {
          const float y = dn.template any<kOp == kLogprobsGrad>(x[e]) + dq[i];
          gb[i] = static_cast<T>(x[e] == neg_inf() ? 0.0f : y);
        }
      }
      __syncthreads();  // dq is the next rows'
    }
  }
}

// ---- launches (one unit a type) ----

// Static LDS, bytes (rounded up).
template <class T, class W, int kC, int kOp>
constexpr int kWaveLds = kOp == kLogprobsTop ? kWaveCandidates * 16 + 512
                         : kOp == kLogprobs  ? 0
                                             : 64 * kWaveEach<T, W, kC> * 4;
constexpr int kRowsLds = 8 * 1024;

struct Launch {
  Rows a;
  Parts pt;
  int waves;       // 0: k_tiny
  int wave;        // k_wave: what it holds in units of 512 bytes, 0: k_rows
  int chunks;      // a lane of k_rows
  bool streamed;   // k_rows: see kStream
  unsigned lds;    // dynamic, bytes
  hipStream_t stream;
};

template <class T>
struct Kernels {
  static void rows(const Launch& c, int op, const LogprobArgs& g);
  static void rows(const Launch& c, const LogprobGradArgs& g);
  static void rows(const Launch& c, int op, const DistillArgs& g);
  static void join(const Launch& c, bool loss, const JoinArgs& g);
};

}  // namespace osp

#endif  // OS_POLICY_H_
