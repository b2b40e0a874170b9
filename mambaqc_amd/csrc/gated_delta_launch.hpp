#pragma once
// Launches of the gated delta rule's kernels (gated_delta.hpp) for one type.
#include "gated_delta.hpp"

namespace mqc {
namespace delta {

#define MQC_BY_KEYS(F)              \
  if (a.k_dim <= 32) return F(32);  \
  if (a.k_dim <= 64) return F(64);  \
  return F(128);

// Columns of the state to a workgroup: 16 as long as the card has room for more workgroups, which is one to a CU
// (of eight waves, or of four for fp32's 128 keys, whose operands leave no registers for it), and two where the
// registers of two fit. 384 walks of 16 columns over 16 chunks, forward and back, us, by 16 and by 32 columns:
//   bf16, 128 keys 73 + 72, 78 + 82;  64 keys 52 + 55, 66 + 66;  32 keys 47 + 52, 64 + 63
//   fp16, 128 keys 113 + 119, 90 + 99;  64 keys 66 + 61, 72 + 69;  32 keys 49 + 52, 65 + 65
//   fp32, 128 keys 139 + 134, 109 + 110;  64 keys 92 + 102, 75 + 82;  32 keys 79 + 87, 69 + 70
// (256 of them: bf16, 128 keys 40 + 38, fp32 68 + 82; 1024: 182 + 182 and 255 + 266.)
template <typename T, int KD>
constexpr bool kTwoToACu = kIn<T> == 1 || (kIn<T> == 2 && KD < 128);
template <typename T, int KD, bool BWD>
int launch_walk(const Args<T>& a, hipStream_t s) {
  const int64_t tiles = a.v_pad / 16, heads = a.batch * a.v_heads;
  constexpr bool kBeside = kIn<T> < 3 || KD < 128;
  if constexpr (kBeside) {
    if (heads * tiles <= 256) {
      const dim3 grid((unsigned)(heads * tiles));
      if constexpr (BWD) delta_bwd_beside_kernel<T, KD><<<grid, dim3(512), 0, s>>>(a);
      else delta_fwd_beside_kernel<T, KD><<<grid, dim3(512), 0, s>>>(a);
      return launch_status();
    }
  }
  if constexpr (!kBeside || kTwoToACu<T, KD>) {
    if (heads * tiles <= (kTwoToACu<T, KD> ? 512 : 256)) {
      const dim3 grid((unsigned)(heads * tiles));
      if constexpr (BWD) delta_bwd_kernel<T, KD, 1><<<grid, dim3(256), 0, s>>>(a);
      else delta_fwd_kernel<T, KD, 1><<<grid, dim3(256), 0, s>>>(a);
      return launch_status();
    }
  }
  const dim3 grid((unsigned)(heads * (tiles / 2)));
  if constexpr (BWD) delta_bwd_kernel<T, KD, 2><<<grid, dim3(256), 0, s>>>(a);
  else delta_fwd_kernel<T, KD, 2><<<grid, dim3(256), 0, s>>>(a);
  return launch_status();
}

template <typename T>
int launch_fwd(const Args<T>& a, hipStream_t s) {
  const unsigned units = (unsigned)(a.batch * a.k_heads * a.chunks);
#define MQC_F(KD)                                                                        \
  [&] {                                                                                  \
    if (units) delta_prep_kernel<T, KD, false><<<dim3(units), dim3(256), 0, s>>>(a);     \
    const int st = launch_status();                                                      \
    return st != MQC_OK ? st : launch_walk<T, KD, false>(a, s);                          \
  }()
  MQC_BY_KEYS(MQC_F)
#undef MQC_F
}

template <typename T>
int launch_bwd(const Args<T>& a, hipStream_t s) {
  const unsigned units = (unsigned)(a.batch * a.k_heads * a.chunks);
  const unsigned parts = (unsigned)(a.batch * a.v_heads * a.chunks);
  const int64_t shares = (a.batch * a.seq * a.k_heads * a.k_dim + 255) / 256;
#define MQC_F(KD)                                                                             \
  [&] {                                                                                       \
    delta_prep_kernel<T, KD, true><<<dim3(units), dim3(256), 0, s>>>(a);                      \
    int st = launch_status();                                                                 \
    if (st == MQC_OK) st = launch_walk<T, KD, true>(a, s);                                    \
    if (st != MQC_OK) return st;                                                              \
    delta_grad_kernel<T, KD><<<dim3(parts), dim3(256 * kGradParts<KD>), 0, s>>>(a);                            \
    if (a.k_heads != a.v_heads)                                                               \
      delta_share_kernel<T><<<dim3((unsigned)(shares < 65536 ? shares : 65536)), dim3(256), 0, s>>>(a); \
    return launch_status();                                                                   \
  }()
  MQC_BY_KEYS(MQC_F)
#undef MQC_F
}

template <typename T>
int launch_step(const Args<T>& a, float* h, hipStream_t s) {
  const unsigned units = (unsigned)(a.batch * a.v_heads * ((a.v_dim + 63) / 64));
#define MQC_F(KD)                                                                    \
  [&] {                                                                              \
    delta_step_kernel<T, KD / 16><<<dim3(units), dim3(256), 0, s>>>(a, h);           \
    return launch_status();                                                          \
  }()
  MQC_BY_KEYS(MQC_F)
#undef MQC_F
}
#undef MQC_BY_KEYS

}  // namespace delta
}  // namespace mqc
