// One AdamW step over many tensors, its states in 32 or in 8 bits, and the gradients' norm that clips
// it. For each element, in fp32 and in this order (no contraction, so that the states do not depend
// on the compiler):
//   g = grad clip;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
//   p = p decay - m / (sqrt(v) root_scale + eps) step_size
// with decay = 1 - lr weight_decay, step_size = lr / (1 - beta1^t), root_scale = 1 / sqrt(1 - beta2^t).
// p is rounded to its type once.
//
// 8-bit states: m and r = sqrt(v) are held as e4m3 numbers times a power of two for each 256 elements,
// the least one that brings the largest of them under 448. Two choices make such a coarse state
// follow its average (a step of e4m3 is 6 to 12 % of the value, an update of v moves it by 5 or by
// 0.1 %, and rounding to nearest would never move it):
//   - a value goes up or down to one of its two neighbours by a number made from its place, the seed
//     and the step t, such that the mean is kept: of m for m, of r^2 = v for r. Over the steps the
//     numbers of one element are a golden-ratio sequence, evenly spread, so the errors of successive
//     steps mostly cancel;
//   - the scale is a power of two, so a value that does not change stays on its code when the scale
//     does not change, and what is rounded is the update alone. (Under a scale that moved with the
//     largest element every element would be rounded anew at each step.)
// r is never rounded to 0 unless it is 0: m / (0 + eps) would be any size. Values that are not finite
// become NaN (code 0x7f), and do not set the scale.
//
// The tensors come as a table in the kernel's arguments (no copy to the device; as many to a launch as
// fit 4 KiB); a workgroup finds its tensor by its place in the running count of workgroups.
//
// All of it is one read and one write of everything, 28 bytes an element with fp32 parameters and
// 32-bit states, 10 with bf16 and 8-bit ones, so a large copy's 5.1 TB/s bounds it: 36 M fp32 parameters
// (1 GB) 163 us; 273 M in bf16 with 8-bit states (2.76 GB) 550 to 560 us step after step, 4.9 to 5.0 TB/s
// (after an idle second the first two 549, then up to 860 at the fifth and back to that within 60, and 560
// where 5 ms lie between them: the card taking up load, not the data); 15 M in fp32 with 8-bit states 45 us. The norm of the 36 M (143 MB) 27 us (one running sum a lane
// instead of four 47).
#include "common.hpp"

namespace mqc {

constexpr int kAdamThreads = 256;
constexpr int kAdamVec = 4;                                  // elements a lane takes at once
constexpr int kAdamIters = 4;                                // and how often, where there are many
constexpr int kAdamChunk = kAdamThreads * kAdamVec * kAdamIters;  // elements of a workgroup then
constexpr int kStateBlock = 256;                             // elements that share a scale

template <int MAX>
struct AdamTableOf {
  static constexpr int kMax = MAX;
  void* p[MAX];
  const void* grad[MAX];
  void* m[MAX];
  void* v[MAX];
  int64_t n[MAX];
  uint32_t first[MAX];  // workgroups before this tensor's
  int count;
};
using AdamTable = AdamTableOf<88>;
struct Adam8Table {
  static constexpr int kMax = 60;
  AdamTableOf<kMax> t;
  float* m_scale[kMax];
  float* v_scale[kMax];
  uint32_t seed[kMax];
};
struct AdamScalars {
  float decay, step_size, root_scale, beta1, one_beta1, beta2, one_beta2, eps;
  const float* clip;
  uint32_t step;
};
static_assert(sizeof(Adam8Table) + sizeof(AdamScalars) <= 4096 &&
                  sizeof(AdamTable) + sizeof(AdamScalars) <= 4096,
              "kernel arguments");

// The tensor of this workgroup: the last that starts at or before it.
__device__ inline int table_find(const uint32_t* first, int count) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= blockIdx.x) lo = mid; else hi = mid;
  }
  return lo;
}

// n <= 4 elements from p, as a vector where that is allowed.
template <typename T>
__device__ inline void load4(const T* p, int n, bool vec, float (&out)[4]) {
  if (vec) {
    load_vec<T, 4>(p, out);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = i < n ? load_scalar(p + i) : 0.f;
  }
}
template <bool STREAM, typename T>
__device__ inline void store4(T* p, int n, bool vec, const float (&in)[4]) {
  if (vec) {
    store_vec<T, 4, STREAM>(p, in);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) store_scalar(p + i, in[i]);
  }
}

// STREAM: for more than the caches hold (mqc_adamw_step), stores that leave no copy there, and sixteen
// elements a lane; else four, for more workgroups.
template <bool STREAM>
constexpr int kAdamTurns = STREAM ? kAdamIters : 1;
template <typename T, bool STREAM>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(AdamTable tab, AdamScalars k) {
#pragma clang fp contract(off)
  constexpr int TURNS = kAdamTurns<STREAM>;
  const int i = table_find(tab.first, tab.count);
  T* p = (T*)tab.p[i];
  const T* grad = (const T*)tab.grad[i];
  float *m = (float*)tab.m[i], *v = (float*)tab.v[i];
  const int64_t n = tab.n[i];
  const int64_t base = (int64_t)(blockIdx.x - tab.first[i]) * (kAdamThreads * kAdamVec * TURNS) +
                       threadIdx.x * kAdamVec;
  const bool fits = (((uintptr_t)p | (uintptr_t)grad) % (4 * sizeof(T)) | ((uintptr_t)m | (uintptr_t)v) % 16) == 0;
  const float clip = k.clip ? *k.clip : 1.f;
  float pv[TURNS][4], gv[TURNS][4], mv[TURNS][4], vv[TURNS][4];
#pragma unroll
  for (int j = 0; j < TURNS; ++j) {
    const int64_t at = base + j * kAdamThreads * kAdamVec;
    const int left = n - at < 4 ? (int)(n - at) : 4;
    const bool vec = fits && left == 4;
    if (left <= 0) continue;
    load4<T>(p + at, left, vec, pv[j]);
    load4<T>(grad + at, left, vec, gv[j]);
    load4<float>(m + at, left, vec, mv[j]);
    load4<float>(v + at, left, vec, vv[j]);
  }
#pragma unroll
  for (int j = 0; j < TURNS; ++j) {
    const int64_t at = base + j * kAdamThreads * kAdamVec;
    const int left = n - at < 4 ? (int)(n - at) : 4;
    const bool vec = fits && left == 4;
    if (left <= 0) continue;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float g = k.clip ? gv[j][c] * clip : gv[j][c];
      mv[j][c] = mv[j][c] * k.beta1 + g * k.one_beta1;
      vv[j][c] = vv[j][c] * k.beta2 + g * g * k.one_beta2;
      pv[j][c] = pv[j][c] * k.decay - mv[j][c] / (sqrtf(vv[j][c]) * k.root_scale + k.eps) * k.step_size;
    }
    store4<STREAM>(p + at, left, vec, pv[j]);
    store4<STREAM>(m + at, left, vec, mv[j]);
    store4<STREAM>(v + at, left, vec, vv[j]);
  }
}

// The largest of a row of 16 lanes, the same in each. Bits of floats >= 0 order as the floats do.
__device__ inline uint32_t row_max_bits(uint32_t v) {
#define MQC_MAX(MOVE)                                                   \
  {                                                                     \
    const uint32_t o = __float_as_uint(MOVE(__uint_as_float(v)));       \
    v = v > o ? v : o;                                                  \
  }
  MQC_MAX(lane_xor1) MQC_MAX(lane_xor2) MQC_MAX(row_rot4) MQC_MAX(row_rot8)
#undef MQC_MAX
  return v;
}

// The exponent field of the block's power of two, from its largest value's bits.
__device__ inline int scale_field(uint32_t top) {
  const int e = (int)(top >> 23) + ((top & 0x7fffff) > 0x600000) - 8;
  return e < 1 ? 1 : e;
}

constexpr uint32_t kMulA = 0x6a09e667u, kMulB = 0xbb67ae85u, kGolden = 0x9e3779b9u;
// An even 32-bit value for an element: sums and products with the fractional parts of sqrt 2, sqrt 3
// and the golden ratio, shifted together.
__device__ inline uint32_t place_bits(uint32_t x) {
  x = (x ^ (x >> 16)) * kMulA;
  x = (x ^ (x >> 15)) * kMulB;
  return x ^ (x >> 16);
}

// 16 consecutive elements from wherever they start.
template <typename T>
__device__ inline void load16(const T* p, int left, float (&out)[16]) {
  typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
  constexpr int EACH = 16 / sizeof(T);
  if (left == 16) {
#pragma unroll
    for (int i = 0; i < 16 / EACH; ++i) {
      const words4 v = reinterpret_cast<const words4*>(p)[i];
#pragma unroll
      for (int c = 0; c < EACH; ++c)
        if constexpr (sizeof(T) == 4) out[EACH * i + c] = __uint_as_float(v[c]);
        else out[EACH * i + c] = io<T>::bits_to_f32(c & 1 ? v[c / 2] >> 16 : v[c / 2] & 0xffffu);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 16; ++c) out[c] = c < left ? load_scalar(p + c) : 0.f;
  }
}
template <typename T>
__device__ inline void store16(T* p, int left, const float (&in)[16]) {
  typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
  if (left == 16) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) {
      words4 v;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if constexpr (sizeof(T) == 4) v[c] = __float_as_uint(in[4 * i + c]);
        else v[c] = pack2<T>(in[8 * i + 2 * c], in[8 * i + 2 * c + 1]);
      reinterpret_cast<words4*>(p)[i] = v;
    }
  } else {
#pragma unroll
    for (int c = 0; c < 16; ++c)
      if (c < left) store_scalar(p + c, in[c]);
  }
}
typedef uint32_t codes16 __attribute__((ext_vector_type(4), aligned(1)));
__device__ inline codes16 load_codes(const uint8_t* p, int left) {
  codes16 v = {0, 0, 0, 0};
  if (left == 16) return *reinterpret_cast<const codes16*>(p);
#pragma unroll
  for (int c = 0; c < 16; ++c)
    if (c < left) v[c / 4] |= (uint32_t)p[c] << (8 * (c % 4));
  return v;
}
__device__ inline void store_codes(uint8_t* p, int left, codes16 v) {
  if (left == 16) {
    *reinterpret_cast<codes16*>(p) = v;
  } else {
#pragma unroll
    for (int c = 0; c < 16; ++c)
      if (c < left) p[c] = (uint8_t)(v[c / 4] >> (8 * (c % 4)));
  }
}
__device__ inline void decode16(codes16 v, float scale, float (&out)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(v[i], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(v[i], true);
    out[4 * i] = lo[0] * scale, out[4 * i + 1] = lo[1] * scale;
    out[4 * i + 2] = hi[0] * scale, out[4 * i + 3] = hi[1] * scale;
  }
}

// The codes of one element's |m| and r under scales of exponent fields mf and vf, rounded by `bits`.
// In steps of its binade (the lowest is 2^-6 on) a value is q; |m| goes up with probability q - floor(q),
// r with (q^2 - k^2) / ((k + 1)^2 - k^2), k = floor(q).
struct AdamCodes { uint32_t m, r; };
__device__ inline AdamCodes adam_codes(float am, float r, int mf, int vf, uint32_t bits, uint32_t step) {
#pragma clang fp contract(off)
  const float um = (float)((bits + step * kGolden) >> 8);  // 2^24 times a number below 1
  const float uv = (float)((((bits << 16) | (bits >> 16)) + step * kMulB) >> 8);
  AdamCodes out;
  {
    const int e = (int)(__float_as_uint(am) >> 23), t = e > mf - 6 ? e : mf - 6;
    const float q = __builtin_ldexpf(am, 130 - t);
    const uint32_t code = ((uint32_t)(t + 6 - mf) << 3) + (uint32_t)fmaf(um, 0x1p-24f, q);
    out.m = code > 0x7eu ? 0x7eu : code;  // q + um may round up to the step past 448
  }
  {
    const int e = (int)(__float_as_uint(r) >> 23), t = e > vf - 6 ? e : vf - 6;
    const float q = __builtin_ldexpf(r, 130 - t), k = floorf(q);
    const bool up = uv * fmaf(k, 0x1p-23f, 0x1p-24f) < (q - k) * (q + k);
    const uint32_t code = ((uint32_t)(t + 6 - vf) << 3) + (uint32_t)k + (up ? 1u : 0u);
    out.r = code > 0 ? code : 1u;
  }
  return out;
}

// A lane takes 16 elements and a row of 16 lanes a block, so the block's largest come from four moves
// within the row. What bounds it is arithmetic more than memory (10 bytes an element with bf16
// parameters): square root and reciprocal are the hardware's with one correction (the root's makes it
// the rounded one), good from 2^-96 to 2^126. Blocks that hold anything else (v of 0, overflow, NaN, a
// scale at the end of its range) take the library's, and tests.
template <typename T>
__global__ __launch_bounds__(kAdamThreads) void adamw8_kernel(Adam8Table tab, AdamScalars k) {
#pragma clang fp contract(off)
  const int i = table_find(tab.t.first, tab.t.count);
  T* p = (T*)tab.t.p[i];
  const T* grad = (const T*)tab.t.grad[i];
  uint8_t *m = (uint8_t*)tab.t.m[i], *v = (uint8_t*)tab.t.v[i];
  const int64_t n = tab.t.n[i];
  const float clip = k.clip ? *k.clip : 1.f;
  const int64_t block = (int64_t)(blockIdx.x - tab.t.first[i]) * (kAdamChunk / kStateBlock) + (threadIdx.x >> 4);
  const int64_t at = block * kStateBlock + (threadIdx.x & 15) * 16;
  if (block * kStateBlock >= n) return;  // whole rows of lanes
  const int left = n - at >= 16 ? 16 : n > at ? (int)(n - at) : 0;
  float pv[16], mm[16], x[16];
  {
    float gv[16];
    load16<T>(grad + at, left, gv);
    const codes16 mc = load_codes(m + at, left), vc = load_codes(v + at, left);
    const float ms = tab.m_scale[i][block], vs = tab.v_scale[i][block];
    load16<T>(p + at, left, pv);
    decode16(mc, ms, mm);
    decode16(vc, vs, x);
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const float g = k.clip ? gv[c] * clip : gv[c];
      mm[c] = mm[c] * k.beta1 + g * k.one_beta1;
      x[c] = x[c] * x[c] * k.beta2 + g * g * k.one_beta2;
    }
  }
  uint32_t mtop = 0, xtop = 0, low = 0xffffffffu;
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const uint32_t ma = __float_as_uint(mm[c]) & 0x7fffffffu, xb = __float_as_uint(x[c]);
    mtop = ma > mtop ? ma : mtop;
    xtop = xb > xtop ? xb : xtop;
    low = xb < low ? xb : low;
  }
  mtop = row_max_bits(mtop);
  xtop = row_max_bits(xtop);
  const bool plain = low >= 0x0f800000u && xtop < 0x7e800000u && mtop < 0x7f800000u && mtop >= 0x08000000u;
  const auto root = [](float a) {
    const float y = __builtin_amdgcn_rsqf(a), s = a * y;
    return fmaf(fmaf(-s, s, a), 0.5f * y, s);
  };
  const uint32_t at_bits = (uint32_t)at + (uint32_t)((uint64_t)at >> 32) * kMulB + tab.seed[i] * kGolden;
  codes16 mo = {0, 0, 0, 0}, vo = {0, 0, 0, 0};
  int mf, vf;
  if (__all(plain)) {
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      x[c] = root(x[c]);
      const float by = __builtin_amdgcn_rcpf(fmaf(x[c], k.root_scale, k.eps));
      pv[c] = fmaf(pv[c], k.decay, -(mm[c] * k.step_size * by));
    }
    store16<T>(p + at, left, pv);
    mf = scale_field(mtop), vf = scale_field(__float_as_uint(root(__uint_as_float(xtop))));
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const AdamCodes code = adam_codes(fabsf(mm[c]), x[c], mf, vf, place_bits(at_bits + c), k.step);
      mo[c / 4] |= (code.m | (__float_as_uint(mm[c]) >> 24 & 0x80u)) << (8 * (c % 4));
      vo[c / 4] |= code.r << (8 * (c % 4));
    }
  } else {
    mtop = xtop = 0;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      x[c] = sqrtf(x[c]);
      pv[c] = pv[c] * k.decay - mm[c] / (x[c] * k.root_scale + k.eps) * k.step_size;
      const uint32_t ma = __float_as_uint(mm[c]) & 0x7fffffffu, xb = __float_as_uint(x[c]);
      if (ma < 0x7f800000u && ma > mtop) mtop = ma;
      if (xb < 0x7f800000u && xb > xtop) xtop = xb;
    }
    store16<T>(p + at, left, pv);
    mf = scale_field(row_max_bits(mtop)), vf = scale_field(row_max_bits(xtop));
    const float mi = __uint_as_float((uint32_t)(254 - mf) << 23);
    const float vi = __uint_as_float((uint32_t)(254 - vf) << 23);
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const bool m_ok = fabsf(mm[c]) < __builtin_inff(), r_ok = x[c] < __builtin_inff();
      const float am = m_ok ? fabsf(mm[c]) * mi : 0.f, r = r_ok ? x[c] * vi : 0.f;
      AdamCodes code = adam_codes(am, r, 127, 127, place_bits(at_bits + c), k.step);
      if (!(r > 0.f)) code.r = 0;
      if (!m_ok) code.m = 0x7f;
      if (!r_ok) code.r = 0x7f;
      mo[c / 4] |= (code.m | (mm[c] < 0.f ? 0x80u : 0u)) << (8 * (c % 4));
      vo[c / 4] |= code.r << (8 * (c % 4));
    }
  }
  if ((threadIdx.x & 15) == 0) {
    tab.m_scale[i][block] = __uint_as_float((uint32_t)mf << 23);
    tab.v_scale[i][block] = __uint_as_float((uint32_t)vf << 23);
  }
  store_codes(m + at, left, mo);
  store_codes(v + at, left, vo);
}

// ---------------------------------------------------------------------------
// The norm: each workgroup's sum of squares in 64 bits (fp32 squares of fp32 gradients neither
// overflow nor lose digits there), then one workgroup's sum of those in a fixed order.
// ---------------------------------------------------------------------------
constexpr int kNormLoads = 8;  // of four elements, a lane
constexpr int kNormChunk = 256 * 4 * kNormLoads;
struct NormTable {
  static constexpr int kMax = 160;
  const void* grad[kMax];
  int64_t n[kMax];
  uint32_t first[kMax];
  int count;
};

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

template <typename T>
__global__ __launch_bounds__(256) void grad_norm_kernel(NormTable tab, double* partial) {
  __shared__ double red[4];
  const int i = table_find(tab.first, tab.count);
  const T* grad = (const T*)tab.grad[i];
  const int64_t n = tab.n[i];
  const int64_t base = (int64_t)(blockIdx.x - tab.first[i]) * kNormChunk + threadIdx.x * 4;
  const bool fits = (uintptr_t)grad % (4 * sizeof(T)) == 0;
  float gv[kNormLoads][4];
#pragma unroll
  for (int j = 0; j < kNormLoads; ++j) {
    const int64_t at = base + j * 1024;
    const int left = n - at < 0 ? 0 : n - at < 4 ? (int)(n - at) : 4;
    load4<T>(grad + at, left, fits && left == 4, gv[j]);
  }
  double part[4] = {};
#pragma unroll
  for (int j = 0; j < kNormLoads; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) part[c] = fma((double)gv[j][c], (double)gv[j][c], part[c]);
  const double s = wave_sum_f64((part[0] + part[1]) + (part[2] + part[3]));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

__global__ __launch_bounds__(1024) void grad_norm_end_kernel(const double* partial, int64_t count,
                                                             double max_norm, float* norm, float* clip) {
  __shared__ double red[16];
  double s = 0;
  for (int64_t i = threadIdx.x; i < count; i += 1024) s += partial[i];
  s = wave_sum_f64(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0;
    for (int i = 0; i < 16; ++i) s += red[i];
    s = sqrt(s);
    *norm = (float)s;
    const double c = max_norm / (s + 1e-6);
    *clip = (float)(c > 1.0 ? 1.0 : c);  // a NaN stays one
  }
}

inline bool known_dtype(int64_t d) { return d == MQC_F32 || d == MQC_BF16 || d == MQC_F16; }

template <typename T>
void launch_adamw(const AdamTable& t, const AdamScalars& k, uint32_t blocks, bool stream, hipStream_t s) {
  if (stream) adamw_kernel<T, true><<<dim3(blocks), dim3(kAdamThreads), 0, s>>>(t, k);
  else adamw_kernel<T, false><<<dim3(blocks), dim3(kAdamThreads), 0, s>>>(t, k);
}
template <typename T>
void launch_adamw(const Adam8Table& t, const AdamScalars& k, uint32_t blocks, hipStream_t s) {
  adamw8_kernel<T><<<dim3(blocks), dim3(kAdamThreads), 0, s>>>(t, k);
}
template <typename T>
void launch_norm(const NormTable& t, double* partial, uint32_t blocks, hipStream_t s) {
  grad_norm_kernel<T><<<dim3(blocks), dim3(256), 0, s>>>(t, partial);
}
#define MQC_LAUNCH(F, dtype, ...)                     \
  switch (dtype) {                                    \
    case MQC_F32: F<float>(__VA_ARGS__); break;       \
    case MQC_BF16: F<bf16_t>(__VA_ARGS__); break;     \
    default: F<f16_t>(__VA_ARGS__); break;            \
  }

// Workgroups of a tensor; a launch (of 256 threads each) holds at most kMaxBlocks of them.
constexpr int64_t kMaxBlocks = 0xffffffffLL / 256;
inline int64_t chunks_of(int64_t n, int64_t chunk) { return (n + chunk - 1) / chunk; }

// Fills tables with the tensors of one dtype after another and calls launch(table, blocks, dtype) for
// each full one. rows: `width` values a tensor, its element count at `n_at` and dtype code at `d_at`.
template <typename Table, typename Put, typename Launch>
int by_tables(const int64_t* rows, int64_t count, int width, int n_at, int d_at, int64_t chunk,
              Put put, Launch launch) {
  for (int dtype : {MQC_F32, MQC_BF16, MQC_F16}) {
    Table t{};
    int used = 0;
    int64_t blocks = 0;
    for (int64_t i = 0; i <= count; ++i) {
      const int64_t* row = rows + i * width;
      const bool mine = i < count && row[d_at] == dtype && row[n_at] > 0;
      const int64_t more = mine ? chunks_of(row[n_at], chunk) : 0;
      if (used > 0 && (i == count || (mine && (used == Table::kMax || blocks + more > kMaxBlocks)))) {
        launch(t, used, (uint32_t)blocks, dtype);
        const int st = launch_status();
        if (st != MQC_OK) return st;
        used = 0, blocks = 0;
      }
      if (mine) put(t, used++, row, (uint32_t)blocks), blocks += more;
    }
  }
  return MQC_OK;
}

inline int check_rows(const int64_t* rows, int64_t count, int width, int pointers, int n_at, int d_at,
                      int64_t chunk) {
  if (count < 0) return MQC_E_SHAPE;
  if (count > 0 && !rows) return MQC_E_NULL;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t* row = rows + i * width;
    if (row[n_at] < 0) return MQC_E_SHAPE;
    if (!known_dtype(row[d_at])) return MQC_E_DTYPE;
    if (chunks_of(row[n_at], chunk) > kMaxBlocks) return MQC_E_LIMIT;
    const uintptr_t size = row[d_at] == MQC_F32 ? 4 : 2;
    for (int c = 0; c < pointers; ++c) {
      if (row[n_at] > 0 && !row[c]) return MQC_E_NULL;
      if (c < 2 && (uintptr_t)row[c] % size) return MQC_E_ALIGN;
    }
  }
  return MQC_OK;
}

template <typename Table>
inline void put_adam(Table& t, int at, const int64_t* row, int64_t n, uint32_t first) {
  t.p[at] = (void*)row[0];
  t.grad[at] = (const void*)row[1];
  t.m[at] = (void*)row[2];
  t.v[at] = (void*)row[3];
  t.n[at] = n;
  t.first[at] = first;
}

}  // namespace mqc

using namespace mqc;

extern "C" int mqc_adamw_step(const int64_t* tensors, int64_t count, float decay, float step_size,
                              float root_scale, float beta1, float one_minus_beta1, float beta2,
                              float one_minus_beta2, float eps, const float* clip, void* stream) {
  const int st = check_rows(tensors, count, 6, 4, 4, 5, kAdamChunk);
  if (st != MQC_OK) return st;
  for (int64_t i = 0; i < count; ++i)
    if ((tensors[6 * i + 2] | tensors[6 * i + 3]) % 4) return MQC_E_ALIGN;
  const AdamScalars k{decay, step_size, root_scale, beta1, one_minus_beta1, beta2, one_minus_beta2,
                      eps, clip, 0};
  // 36 M fp32 parameters (1 GB) 164 us streamed, 177 not; what fits the 256 MiB cache is found there at
  // the next step. Of a small step, sixteen elements a lane leave workgroups too few: 2.2 M fp32
  // parameters 11.3 us, or 9.6 with four, 16 M in bf16 57 and 53; 36 M 163 and 165, and their norm, whose
  // gradients the cache then holds no longer, 27 and 45.
  int64_t bytes = 0;
  for (int64_t i = 0; i < count && bytes <= 256LL << 20; ++i)
    bytes += tensors[6 * i + 4] * (tensors[6 * i + 5] == MQC_F32 ? 16 : 12);
  const bool many = bytes > 256LL << 20;
  const int64_t chunk = kAdamThreads * kAdamVec * (many ? kAdamTurns<true> : kAdamTurns<false>);
  return by_tables<AdamTable>(
      tensors, count, 6, 4, 5, chunk,
      [](AdamTable& t, int at, const int64_t* row, uint32_t first) { put_adam(t, at, row, row[4], first); },
      [&](AdamTable& t, int used, uint32_t blocks, int dtype) {
        t.count = used;
        MQC_LAUNCH(launch_adamw, dtype, t, k, blocks, many, (hipStream_t)stream)
      });
}

extern "C" int mqc_adamw8_step(const int64_t* tensors, int64_t count, float decay, float step_size,
                               float root_scale, float beta1, float one_minus_beta1, float beta2,
                               float one_minus_beta2, float eps, const float* clip, uint32_t step,
                               void* stream) {
  const int st = check_rows(tensors, count, 9, 6, 6, 7, kAdamChunk);
  if (st != MQC_OK) return st;
  for (int64_t i = 0; i < count; ++i)
    if ((tensors[9 * i + 4] | tensors[9 * i + 5]) % 4) return MQC_E_ALIGN;
  const AdamScalars k{decay, step_size, root_scale, beta1, one_minus_beta1, beta2, one_minus_beta2,
                      eps, clip, step};
  return by_tables<Adam8Table>(
      tensors, count, 9, 6, 7, kAdamChunk,
      [](Adam8Table& t, int at, const int64_t* row, uint32_t first) {
        put_adam(t.t, at, row, row[6], first);
        t.m_scale[at] = (float*)row[4];
        t.v_scale[at] = (float*)row[5];
        t.seed[at] = (uint32_t)row[8];
      },
      [&](Adam8Table& t, int used, uint32_t blocks, int dtype) {
        t.t.count = used;
        MQC_LAUNCH(launch_adamw, dtype, t, k, blocks, (hipStream_t)stream)
      });
}

extern "C" int64_t mqc_grad_norm_workspace_bytes(const int64_t* tensors, int64_t count) {
  const int st = check_rows(tensors, count, 3, 1, 1, 2, kNormChunk);
  if (st != MQC_OK) return st;
  int64_t blocks = 0;
  for (int64_t i = 0; i < count; ++i) blocks += chunks_of(tensors[3 * i + 1], kNormChunk);
  return blocks * (int64_t)sizeof(double);
}

extern "C" int mqc_grad_norm(const int64_t* tensors, int64_t count, double max_norm, float* norm,
                             float* clip, void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t need = mqc_grad_norm_workspace_bytes(tensors, count);
  if (need < 0) return (int)need;
  if (!norm || !clip) return MQC_E_NULL;
  if (workspace_bytes < need) return MQC_E_SPACE;
  if (need > 0 && !workspace) return MQC_E_NULL;
  if (!aligned(workspace, 8)) return MQC_E_ALIGN;
  double* partial = (double*)workspace;
  hipStream_t s = (hipStream_t)stream;
  const int st = by_tables<NormTable>(
      tensors, count, 3, 1, 2, kNormChunk,
      [](NormTable& t, int at, const int64_t* row, uint32_t first) {
        t.grad[at] = (const void*)row[0];
        t.n[at] = row[1];
        t.first[at] = first;
      },
      [&](NormTable& t, int used, uint32_t blocks, int dtype) {
        t.count = used;
        MQC_LAUNCH(launch_norm, dtype, t, partial, blocks, s)
        partial += blocks;
      });
  if (st != MQC_OK) return st;
  grad_norm_end_kernel<<<dim3(1), dim3(1024), 0, s>>>((const double*)workspace,
                                                      need / (int64_t)sizeof(double), max_norm, norm, clip);
  return launch_status();
}
