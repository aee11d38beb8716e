// Instantiates the policy kernels (os_policy.h) for one element type.
#ifndef OS_POLICY_LAUNCH_H_
#define OS_POLICY_LAUNCH_H_

#include <algorithm>

#include "os_policy.h"

namespace osp {

constexpr int kCus = 256;

// Waves of a kernel that fit a SIMD by its registers (512 a lane, in eights).
template <auto kKernel>
int waves_per_simd() {
  static const int n = [] {
    hipFuncAttributes f;
    if (hipFuncGetAttributes(&f, reinterpret_cast<const void*>(kKernel)) != hipSuccess) return 4;
    return std::max(1, std::min(8, 512 / std::max(8, (f.numRegs + 7) / 8 * 8)));
  }();
  return n;
}

// A workgroup goes over several rows (loading the next one early) once the
// card is full: as many as are resident, the rounds evened out.
inline dim3 row_grid(const Launch& c, int per_simd, int lds) {
  int blocks = std::max(1, 4 * per_simd / c.waves);
  if (lds > 0) blocks = std::max(1, std::min(blocks, 160 * 1024 / lds));
  const int64_t most = std::max<int64_t>(1, int64_t{kCus} * blocks / c.pt.parts);
  const int64_t rounds = (c.a.n + most - 1) / most;
  return dim3(static_cast<unsigned>((c.a.n + rounds - 1) / rounds), static_cast<unsigned>(c.pt.parts));
}

template <class T, int kOp, class G>
void launch_rows(const Launch& c, const G& g) {
  if (c.waves == 0) {
    const int64_t blocks = std::min<int64_t>((c.a.n + kTinyRows - 1) / kTinyRows, kCus * 8);
    hipLaunchKernelGGL((k_tiny<T, kOp>), dim3(static_cast<unsigned>(blocks)), dim3(kTinyBlock), 0,
                       c.stream, c.a, g);
    return;
  }
  if (c.wave != 0) {
    const auto go = [&](auto mask, auto chunk, auto chunks) {
      using W = decltype(chunk);
      constexpr bool kMask = decltype(mask)::value;
      constexpr int kC = decltype(chunks)::value;
      constexpr auto kernel = &k_wave<T, kMask, W, kC, kOp>;
      hipLaunchKernelGGL(kernel, row_grid(c, waves_per_simd<kernel>(), kWaveLds<T, W, kC, kOp>),
                         dim3(64), 0, c.stream, c.a, g);
    };
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    constexpr std::integral_constant<int, 3> three;
    constexpr std::integral_constant<int, 4> four;
    [[maybe_unused]] constexpr std::integral_constant<int, 6> six;
    [[maybe_unused]] constexpr std::integral_constant<int, 8> eight;
    const auto by_chunks = [&](auto mask) {
      switch (c.wave) {
        case 1: return go(mask, u32x2{}, one);
        case 2: return go(mask, u32x4{}, one);
        case 3: return go(mask, u32x2{}, three);
        case 4: return go(mask, u32x4{}, two);
        case 6: return go(mask, u32x4{}, three);
        case 8: return go(mask, u32x4{}, four);
        default:
          if constexpr (sizeof(T) == 4) {
            if (c.wave == 12) go(mask, u32x4{}, six);
            else go(mask, u32x4{}, eight);
          }
      }
    };
    if (c.a.legal != nullptr) by_chunks(std::true_type{});
    else by_chunks(std::false_type{});
    return;
  }
  const auto go = [&](auto mask, auto chunks, auto stream) {
    constexpr auto kernel =
        &k_rows<T, decltype(mask)::value, decltype(chunks)::value, kOp, decltype(stream)::value>;
    hipLaunchKernelGGL(kernel, row_grid(c, waves_per_simd<kernel>(), static_cast<int>(c.lds) + kRowsLds),
                       dim3(64 * c.waves), c.lds, c.stream, c.a, c.pt, g);
  };
  constexpr std::integral_constant<int, kFewChunks> few;
  constexpr std::integral_constant<int, kMidChunks> mid;
  constexpr std::integral_constant<int, kChunks> many;
  constexpr std::true_type yes;
  constexpr std::false_type no;
  if (c.a.legal != nullptr) {
    if (c.chunks == few) go(yes, few, no);
    else go(yes, mid, no);
  } else {
    if (c.chunks == few) go(no, few, no);
    else if (c.chunks == mid) go(no, mid, no);
    else if (c.streamed) go(no, many, yes);
    else go(no, many, no);
  }
}

template <class T>
void Kernels<T>::rows(const Launch& c, int op, const LogprobArgs& g) {
  if (op == kLogprobs) launch_rows<T, kLogprobs>(c, g);
  else launch_rows<T, kLogprobsTop>(c, g);
}
template <class T>
void Kernels<T>::rows(const Launch& c, const LogprobGradArgs& g) {
  launch_rows<T, kLogprobsGrad>(c, g);
}
template <class T>
void Kernels<T>::rows(const Launch& c, int op, const DistillArgs& g) {
  if (op == kDistill) launch_rows<T, kDistill>(c, g);
  else if (op == kDistillFused) launch_rows<T, kDistillFused>(c, g);
  else launch_rows<T, kDistillGrad>(c, g);
}
template <class T>
void Kernels<T>::join(const Launch& c, bool loss, const JoinArgs& g) {
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(c.a.n, kJoinGridX)),
                  static_cast<unsigned>((c.a.n + kJoinGridX - 1) / kJoinGridX));
  if (loss) hipLaunchKernelGGL((k_join<T, true>), grid, dim3(kJoin), 0, c.stream, c.a, g);
  else hipLaunchKernelGGL((k_join<T, false>), grid, dim3(kJoin), 0, c.stream, c.a, g);
}

}  // namespace osp

#endif  // OS_POLICY_LAUNCH_H_
