// Instantiates the policy kernels (os_policy.h) for one element type.
#ifndef OS_POLICY_LAUNCH_H_
#define OS_POLICY_LAUNCH_H_

#include "os_policy.h"

namespace osp {

template <class T, int kOp, class G>
void launch_rows(const Launch& c, const G& g) {
  if (c.waves == 0) {
    hipLaunchKernelGGL((k_tiny<T, kOp>), c.grid, dim3(kTinyBlock), 0, c.stream, c.a, g);
    return;
  }
  if (c.wave != 0) {
    const auto go = [&](auto mask) {
      constexpr bool kMask = decltype(mask)::value;
      if (c.wave == 1)
        hipLaunchKernelGGL((k_wave<T, kMask, 1, kOp>), c.grid, dim3(64), 0, c.stream, c.a, g);
      else if (c.wave == 2)
        hipLaunchKernelGGL((k_wave<T, kMask, 2, kOp>), c.grid, dim3(64), 0, c.stream, c.a, g);
      else
        hipLaunchKernelGGL((k_wave<T, kMask, 4, kOp>), c.grid, dim3(64), 0, c.stream, c.a, g);
    };
    if (c.a.legal != nullptr) go(std::true_type{});
    else go(std::false_type{});
    return;
  }
  const dim3 block(64 * c.waves);
  const auto go = [&](auto mask, auto chunks) {
    hipLaunchKernelGGL((k_rows<T, decltype(mask)::value, decltype(chunks)::value, kOp>), c.grid,
                       block, c.lds, c.stream, c.a, c.pt, g);
  };
  constexpr std::integral_constant<int, kFewChunks> few;
  constexpr std::integral_constant<int, kMidChunks> mid;
  constexpr std::integral_constant<int, kChunks> many;
  if (c.a.legal != nullptr) {
    if (c.chunks == few) go(std::true_type{}, few);
    else go(std::true_type{}, mid);
  } else {
    if (c.chunks == few) go(std::false_type{}, few);
    else if (c.chunks == mid) go(std::false_type{}, mid);
    else go(std::false_type{}, many);
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
  if (loss) hipLaunchKernelGGL((k_join<T, true>), c.grid, dim3(kJoin), 0, c.stream, c.a, g);
  else hipLaunchKernelGGL((k_join<T, false>), c.grid, dim3(kJoin), 0, c.stream, c.a, g);
}

}  // namespace osp

#endif  // OS_POLICY_LAUNCH_H_
