// C-ABI of the policy operators (include/os_mcts.h, "Policy operators"):
// argument checks, the choice of kernel and workgroup for a call's rows, and
// the launches.  The kernels are os_policy.h's.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "os_error.h"
#include "os_policy.h"

namespace osx {
namespace {

using namespace osp;

constexpr int kCus = 256;
constexpr int64_t kKib = 1024;
constexpr int64_t kLastLevelCache = int64_t{256} << 20;
// (sums_plan leaves rows that fit a workgroup whole, masked or not)
constexpr int64_t kWholeRow = kMaxWaves * kMidChunks * kKib;
static_assert(OS_AZ_NO_WORKSPACE_ACTIONS * 4 <= kWholeRow);

// ---- how the workgroups share the rows ----

struct Plan {
  int waves;  // 0: k_tiny
  int wave;   // k_wave: what it holds in units of 512 bytes, 0: k_rows
  int chunks;  // a lane of k_rows
  bool streamed;  // k_rows does not ask the caches to keep the logits
  Parts pt;
};

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Parts of a multiple of 64 actions.  The last one is never below 64: `parts`
// is chosen with at least 4096 actions each and at most 64 of them, or with
// 8192 and at most 128, so rounding the others up leaves the last at least
// 4096 - 63 * 63 (8192 - 127 * 63).
Parts split(int32_t v, int64_t parts) {
  Parts p;
  p.part = parts <= 1 ? v : static_cast<int32_t>(up(up(v, parts), 64) * 64);
  p.parts = static_cast<int32_t>(up(v, p.part));
  return p;
}

// Rows of up to kWaveMax actions: 16 lanes or a wave each.
bool short_rows(const Rows& a, int size, Plan* p) {
  const int64_t bytes = int64_t{a.v} * size;
  if (a.v > kWaveMax) return false;
  p->pt = Parts{1, a.v};
  if (a.v <= kTinyMax) return true;
  p->waves = 1;
  const int units = static_cast<int>(up(bytes, 512));
  p->wave = units <= 4 ? units : units <= 6 ? 6 : units <= 8 ? 8 : units <= 12 ? 12 : 16;
  return true;
}

// Bytes a wave of k_rows holds: 64 lanes x 16 a chunk.
int64_t wave_bytes(const Rows& a) { return (a.legal ? kMidChunks : kChunks) * kKib; }

// Chunks a lane and waves for `bytes` a workgroup: with `wide` as many waves as
// a workgroup has (few rows: each is over sooner), else eight chunks as long as
// they do (4194 x 16000 f32, loss and gradient: 146 us in four, 123 in eight, 136
// in sixteen).  Logits beyond the last-level cache want fewer, longer waves and
// no place in the cache, once rows fill them (1 GiB of f32, loss and gradient:
// rows of 32768 445 us in eight, 425 in sixteen; rows of 4100 515 and 733).
void fit(const Rows& a, int size, int64_t bytes, bool wide, Plan* p) {
  const bool cached = a.n * a.v * size <= kLastLevelCache;
  if (wide && bytes <= kMaxWaves * kFewChunks * kKib) p->chunks = kFewChunks;
  else if (a.legal || bytes <= (wide || cached ? kMaxWaves * kMidChunks : 32) * kKib)
    p->chunks = kMidChunks;
  else p->chunks = kChunks;
  p->waves = static_cast<int>(up(bytes, p->chunks * kKib));
  // (16-bit rows that start between dwords share their lines' ends with their
  // neighbours: dropped early, those are read twice - 50021 bf16 actions x 2048
  // rows, log probabilities: 42 us kept, 51 us dropped)
  p->streamed = p->chunks == kChunks && !cached &&
                (size == 4 || ((reinterpret_cast<uintptr_t>(a.x) | (a.ld * size)) & 3) == 0);
}

// Kernels that need the row's sums.
Plan sums_plan(const Rows& a, int size) {
  Plan p{};
  if (short_rows(a, size, &p)) return p;
  const int64_t bytes = int64_t{a.v} * size, most = kMaxWaves * wave_bytes(a);
  // A row in one workgroup as long as it fits: joining parts costs a launch and
  // the gradient a second read.  Only few rows near that limit are over sooner
  // in parts (131072 bf16 actions, top 20: 1 row 13 us in parts, 17 whole; 128
  // rows 22 and 19; 65536 actions: 1 row 12.5 and 12, 256 rows 22 and 14).
  // Rows that do not fit go in parts of 64 KiB, four workgroups a compute unit.
  int64_t parts = bytes <= most ? 1 : up(bytes, 64 * kKib);
  if (a.n <= 64 && bytes > kWholeRow) parts = std::max(parts, bytes / (16 * kKib));
  p.pt = split(a.v, std::min<int64_t>(parts, kMaxSplit));
  fit(a, size, int64_t{p.pt.part} * size, a.n * p.pt.parts < 4 * kCus, &p);
  return p;
}

// Gradients from known sums: parts are free, and small ones overlap better.
Plan grad_plan(const Rows& a, int size) {
  Plan p{};
  if (short_rows(a, size, &p)) return p;
  const int64_t bytes = int64_t{a.v} * size;
  p.pt = split(a.v, up(bytes, 64 * kKib));
  fit(a, size, int64_t{p.pt.part} * size, a.n * p.pt.parts < 4 * kCus, &p);
  return p;
}

int type_size(int dtype) { return dtype == OS_AZ_F32 ? 4 : 2; }

Launch launch(const Rows& a, const Plan& p, void* stream) {
  return Launch{a, p.pt, p.waves, p.wave, p.chunks, p.streamed, 0, static_cast<hipStream_t>(stream)};
}

// Each part's sums and top keys, and the rows' stats where a caller wants none.
int64_t workspace_bytes_of(const Rows& a, const Plan& p, int top) {
  if (p.pt.parts <= 1) return 0;
  return a.n * (p.pt.parts * (static_cast<int64_t>(sizeof(PartSums)) + 8 * int64_t{top}) + 8);
}

// The LDS of k_rows' tables of listed weights: a row's and the next one's.
void target_lds(const Plan& p, DistillArgs* g, Launch* c) {
  if (p.waves == 0 || p.wave != 0) return;
  g->hash = 64;
  while (g->hash < 2 * g->t.k) g->hash *= 2;
  c->lds = static_cast<unsigned>(g->hash) * 24;
}

// ---- argument checks ----

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
  if (p->num_rows > INT32_MAX) return Fail(OS_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
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

template <class F>
int by_dtype(int dtype, F f) {
  if (dtype == OS_AZ_F32) f(Kernels<float>{});
  else if (dtype == OS_AZ_BF16) f(Kernels<__bf16>{});
  else f(Kernels<_Float16>{});
  HIP_TRY(hipGetLastError());
  return OS_OK;
}

int check_workspace(int64_t need, const void* workspace, int64_t bytes) {
  if (need == 0) return OS_OK;
  if (!workspace || bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return Fail(OS_ERR_INVALID, "workspace below os_az_rows_workspace, or not 16-byte aligned");
  return OS_OK;
}

// A call's buffer: `n` rows of `bytes` bytes in elements of `size`, `ld` bytes apart.
struct Buffer {
  const char* name;
  const void* p;
  int64_t n, ld, bytes;
  int size;
  bool out;
};

// The end of the buffer (a stride so large that it leaves 64 bits: of the memory).
uint64_t past(const Buffer& b) {
  uint64_t far, end;
  const uint64_t at = reinterpret_cast<uintptr_t>(b.p);
  if (__builtin_mul_overflow(static_cast<uint64_t>(b.n - 1), static_cast<uint64_t>(b.ld), &far) ||
      __builtin_add_overflow(far, at + static_cast<uint64_t>(b.bytes), &end))
    return UINT64_MAX;
  return end;
}

// Of two buffers whose extents meet: whether they are disjoint columns of one
// buffer's rows.
bool columns(const Buffer& a, const Buffer& b) {
  if (a.ld != b.ld || a.ld == 0) return false;
  const uint64_t a0 = reinterpret_cast<uintptr_t>(a.p), b0 = reinterpret_cast<uintptr_t>(b.p);
  const uint64_t ld = static_cast<uint64_t>(a.ld);
  const uint64_t off = b0 >= a0 ? (b0 - a0) % ld : (ld - (a0 - b0) % ld) % ld;
  return off >= static_cast<uint64_t>(a.bytes) && off + static_cast<uint64_t>(b.bytes) <= ld;
}

// Elements lie at multiples of their size (a row's single values are scalar
// loads, which drop an address's low bits).  Results share no memory with each
// other or with what the call reads: rows are worked on in any order, and some
// operands are read again after a result is written.
template <int kCount>
int check_buffers(const Buffer (&all)[kCount]) {
  uint64_t lo[kCount], hi[kCount];
  for (int i = 0; i < kCount; ++i) {
    const Buffer& a = all[i];
    const bool there = a.p != nullptr && a.n > 0 && a.bytes > 0;
    lo[i] = there ? reinterpret_cast<uintptr_t>(a.p) : UINT64_MAX;
    hi[i] = there ? past(a) : 0;
    if (there && (lo[i] & static_cast<uint64_t>(a.size - 1)))
      return Fail(OS_ERR_INVALID, std::string(a.name) + " not aligned to its type");
  }
  for (int i = 0; i < kCount; ++i) {
    if (!all[i].out) continue;
    for (int j = 0; j < kCount; ++j)
      if (lo[i] < hi[j] && lo[j] < hi[i] && i != j && !columns(all[i], all[j]))
        return Fail(OS_ERR_INVALID, std::string(all[i].name) + " overlaps " + all[j].name);
  }
  return OS_OK;
}

// `each` elements a row, rows end to end.
Buffer per_row(const char* name, const void* p, const Rows& a, int size, int64_t each) {
  return Buffer{name, p, 1, 0, a.n * each * size, size, false};
}
Buffer strided(const char* name, const void* p, const Rows& a, int64_t stride) {
  return Buffer{name, p, a.n, stride * 4, 4, 4, false};
}
Buffer matrix(const char* name, const void* p, const Rows& a, int64_t ld, int64_t columns, int size) {
  return Buffer{name, p, a.n, ld * size, columns * size, size, false};
}
Buffer result(Buffer b) {
  b.out = true;
  return b;
}
Buffer logits_of(const Rows& a, int size) { return matrix("logits", a.x, a, a.ld, a.v, size); }
Buffer legal_of(const Rows& a) { return matrix("legal", a.legal, a, a.lld, a.v, 1); }
Buffer ids_of(const Rows& a, const Target& t) {
  return matrix("target actions", t.ids, a, t.ids_ld, t.k, t.wide ? 8 : 4);
}
Buffer values_of(const Rows& a, const Target& t) {
  const bool half = t.type == OS_AZ_LOGITS_BF16 || t.type == OS_AZ_LOGITS_F16;
  return matrix("target", t.val, a, t.val_ld, t.k, half ? 2 : 4);
}
Buffer workspace_of(const void* p, int64_t bytes) { return Buffer{"workspace", p, 1, 0, bytes, 16, true}; }

// Fail() keeps its message in a string, which may run out of memory: nothing
// leaves a C entry but a code.
template <class F>
auto guarded(F f) -> decltype(f()) {
  try {
    return f();
  } catch (...) {
    return OS_ERR_DEVICE;
  }
}

}  // namespace
}  // namespace osx

using namespace osx;

extern "C" {

int64_t os_az_rows_workspace(const os_az_rows* rows, int32_t top) {
  return guarded([&]() -> int64_t {
    Rows a;
    if (const int rc = check_rows(rows, &a)) return rc;
    if (top < 0 || top > OS_AZ_MAX_TOP) return Fail(OS_ERR_INVALID, "top must be in [0, OS_AZ_MAX_TOP]");
    if (a.n == 0) return 0;
    return workspace_bytes_of(a, sums_plan(a, type_size(rows->dtype)), top);
  });
}

int os_az_logprobs_async(const os_az_rows* rows, const void* actions, int32_t wide,
                         float* logprob, float* entropy, float* stats, int32_t top,
                         int64_t* top_action, float* top_logprob, void* workspace,
                         int64_t workspace_bytes, void* hip_stream) {
  return guarded([&]() -> int {
    Rows a;
    if (const int rc = check_rows(rows, &a)) return rc;
    if (top < 0 || top > OS_AZ_MAX_TOP) return Fail(OS_ERR_INVALID, "top must be in [0, OS_AZ_MAX_TOP]");
    if (a.n == 0) return OS_OK;
    if (!entropy || (top > 0 && (!top_action || !top_logprob)) || (!actions != !logprob))
      return Fail(OS_ERR_INVALID, "null logprobs buffer");
    const Plan p = sums_plan(a, type_size(rows->dtype));
    const int64_t need = workspace_bytes_of(a, p, top);
    if (const int rc = check_workspace(need, workspace, workspace_bytes)) return rc;
    if (const int rc = check_buffers(
            {logits_of(a, type_size(rows->dtype)), legal_of(a), per_row("actions", actions, a, wide ? 8 : 4, 1),
             result(per_row("logprob", logprob, a, 4, 1)), result(per_row("entropy", entropy, a, 4, 1)),
             result(per_row("stats", stats, a, 4, 2)), result(per_row("top_action", top_action, a, 8, top)),
             result(per_row("top_logprob", top_logprob, a, 4, top)), workspace_of(workspace, need)}))
      return rc;
    LogprobArgs g{actions, wide != 0, top, logprob, entropy, stats, top_action, top_logprob,
                  nullptr, nullptr};
    if (need > 0) {
      g.sums = static_cast<PartSums*>(workspace);
      g.part_keys = top > 0 ? reinterpret_cast<uint64_t*>(g.sums + a.n * p.pt.parts) : nullptr;
    }
    return by_dtype(rows->dtype, [&](auto k) {
      Launch c = launch(a, p, hip_stream);
      k.rows(c, top > 0 ? kLogprobsTop : kLogprobs, g);
      if (need == 0) return;
      k.join(c, false, JoinArgs{g, DistillArgs{}, p.pt.parts});
    });
  });
}

int os_az_logprobs_grad_async(const os_az_rows* rows, const void* actions, int32_t wide,
                              const float* entropy, const float* stats, int32_t top,
                              const int64_t* top_action, const float* g_logprob,
                              int64_t g_logprob_stride, const float* g_entropy,
                              int64_t g_entropy_stride, const float* g_top, void* grad,
                              int64_t grad_ld, void* hip_stream) {
  return guarded([&]() -> int {
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
    const int size = type_size(rows->dtype);
    if (const int rc = check_buffers(
            {logits_of(a, size), legal_of(a), per_row("actions", actions, a, wide ? 8 : 4, 1),
             per_row("entropy", g_entropy ? entropy : nullptr, a, 4, 1), per_row("stats", stats, a, 4, 2),
             per_row("top_action", top_action, a, 8, top), strided("g_logprob", g_logprob, a, g_logprob_stride),
             strided("g_entropy", g_entropy, a, g_entropy_stride), per_row("g_top", g_top, a, 4, top),
             result(matrix("grad", grad, a, grad_ld, a.v, size))}))
      return rc;
    const Plan p = grad_plan(a, size);
    const LogprobGradArgs g{actions,    wide != 0,        top,       entropy,          stats,
                            top_action, g_logprob,        g_logprob_stride, g_entropy, g_entropy_stride,
                            g_top,      grad,             grad_ld};
    return by_dtype(rows->dtype, [&](auto k) {
      Launch c = launch(a, p, hip_stream);
      c.lds = p.waves > 0 && p.wave == 0 && top > 0 ? 2 * 128 * 12 : 0;
      k.rows(c, g);
    });
  });
}

int os_az_distill_async(const os_az_rows* rows, const os_az_target* target, const float* weight,
                        float* loss, float* target_entropy, float* stats, void* grad,
                        int64_t grad_ld, void* workspace, int64_t workspace_bytes,
                        void* hip_stream) {
  return guarded([&]() -> int {
    Rows a;
    Target t;
    if (const int rc = check_rows(rows, &a)) return rc;
    if (const int rc = check_target(target, a, &t)) return rc;
    if (grad)
      if (const int rc = check_grad(a, rows->dtype, grad, grad_ld)) return rc;
    if (a.n == 0) return OS_OK;
    if (!loss) return Fail(OS_ERR_INVALID, "null loss");
    const int size = type_size(rows->dtype);
    const Plan p = sums_plan(a, size);
    const int64_t need = workspace_bytes_of(a, p, 0);
    const bool parts = need > 0;
    if (const int rc = check_workspace(need, workspace, workspace_bytes)) return rc;
    if (const int rc = check_buffers(
            {logits_of(a, size), legal_of(a), ids_of(a, t), values_of(a, t),
             per_row("weight", grad ? weight : nullptr, a, 4, 1), result(per_row("loss", loss, a, 4, 1)),
             result(per_row("target_entropy", target_entropy, a, 4, 1)),
             result(per_row("stats", stats, a, 4, 2)), result(matrix("grad", grad, a, grad_ld, a.v, size)),
             workspace_of(workspace, need)}))
      return rc;
    DistillArgs g{t, weight, 1, loss, target_entropy, stats, grad, grad_ld, 0};
    return by_dtype(rows->dtype, [&](auto k) {
      Launch c = launch(a, p, hip_stream);
      if (!parts) {
        if (grad) target_lds(p, &g, &c);
        k.rows(c, grad ? kDistillFused : kDistill, g);
        return;
      }
      LogprobArgs lp{};
      lp.sums = static_cast<PartSums*>(workspace);
      // (the gradient's launch reads the row's sums: left behind the parts')
      if (!stats) g.stats = reinterpret_cast<float*>(lp.sums + a.n * p.pt.parts);
      k.rows(c, kLogprobs, lp);
      k.join(c, true, JoinArgs{lp, g, p.pt.parts});
      if (!grad) return;
      const Plan q = grad_plan(a, size);
      Launch d = launch(a, q, hip_stream);
      target_lds(q, &g, &d);
      k.rows(d, kDistillGrad, g);
    });
  });
}

int os_az_distill_grad_async(const os_az_rows* rows, const os_az_target* target,
                             const float* weight, int64_t weight_stride, const float* stats,
                             void* grad, int64_t grad_ld, void* hip_stream) {
  return guarded([&]() -> int {
    Rows a;
    Target t;
    if (const int rc = check_rows(rows, &a)) return rc;
    if (const int rc = check_target(target, a, &t)) return rc;
    if (weight_stride < 0) return Fail(OS_ERR_INVALID, "negative stride");
    if (const int rc = check_grad(a, rows->dtype, grad, grad_ld)) return rc;
    if (a.n == 0) return OS_OK;
    if (!stats || !grad) return Fail(OS_ERR_INVALID, "null gradient buffer");
    const int size = type_size(rows->dtype);
    if (const int rc = check_buffers({logits_of(a, size), legal_of(a), ids_of(a, t), values_of(a, t),
                                      strided("weight", weight, a, weight_stride),
                                      per_row("stats", stats, a, 4, 2),
                                      result(matrix("grad", grad, a, grad_ld, a.v, size))}))
      return rc;
    const Plan p = grad_plan(a, size);
    DistillArgs g{t, weight, weight_stride, nullptr, nullptr, const_cast<float*>(stats),
                  grad, grad_ld, 0};
    return by_dtype(rows->dtype, [&](auto k) {
      Launch c = launch(a, p, hip_stream);
      target_lds(p, &g, &c);
      k.rows(c, kDistillGrad, g);
    });
  });
}

}  // extern "C"
