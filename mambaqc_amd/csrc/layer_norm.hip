// Layer norm over the last axis, with its gradients:
//   h = (x - mean x) / sqrt(mean (x - mean x)^2 + eps),  y = h w + b
//   dx = (u - mean u - h mean(u h)) / sqrt(..) with u = dy w,  dw = sum over rows of dy h,  db = sum of dy
// (without w it is 1, without b 0). A row stays in the registers of its team of lanes between its loads
// and its store, so the variance is the mean square about the mean that is known by then, and memory
// bounds both directions. Everything between is fp32. 8192 rows of 768 in bf16 take 8.0 us forward and 10.0
// back (25 and 38 MB), with 3.8 for the sums over the workgroups.
#include "common.hpp"

namespace mqc {

constexpr int64_t kLayerNormMaxWidth = 8192;

template <typename T>
struct LayerNormArgs {
  const T* x;
  int64_t x_row;  // elements between rows of x
  const float *w, *b;
  int64_t rows, d;
  float eps;
  T* y;
  float* stats;  // [rows, 2]: mean and 1 / sqrt(..), or NULL
  // backward
  const T* dy;
  T* dx;
  float* part;  // [2, workgroups, d]: sums of dy h and of dy, or NULL
};

// The sum over a team of LANES lanes (16, 32, a wave, or all waves of the workgroup: 0), the same in
// every lane of it. `red` holds 16 floats a sum.
template <int LANES, int N>
__device__ inline void norm_sum(float (&v)[N], float* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (LANES == 16 || LANES == 32) {
      v[i] += lane_xor1(v[i]);
      v[i] += lane_xor2(v[i]);
      v[i] += row_rot4(v[i]);
      v[i] += row_rot8(v[i]);
      if constexpr (LANES == 32) v[i] += __shfl_xor(v[i], 16);
    } else {
      v[i] = wave_sum_all(v[i]);
    }
  }
  if constexpr (LANES == 0) {
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[16 * i + wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll 2
      for (int w = 0; w < waves; ++w) v[i] += red[16 * i + w];
    }
  }
}

template <int LANES>
constexpr int kNormTeams = LANES ? 256 / LANES : 1;

// A lane holds elements 4 (lane + team m) + 0..3 of its row for m < NV. STREAM: stores that leave no copy
// in the caches.
template <typename T, int NV, int LANES, bool STREAM>
__global__ __launch_bounds__(LANES ? 256 : 512) void layer_norm_fwd_kernel(LayerNormArgs<T> k) {
  __shared__ float red[2][LANES ? 1 : 16];
  const int team = LANES ? LANES : blockDim.x, t = LANES ? threadIdx.x % team : threadIdx.x;
  const int d = (int)k.d;
  const int64_t row = (int64_t)blockIdx.x * kNormTeams<LANES> + (LANES ? threadIdx.x / team : 0);
  if (row >= k.rows) return;  // whole teams; a team of several waves has its row
  const T* from = k.x + row * k.x_row;
  float x[NV][4], s[1] = {0.f};
#pragma unroll
  for (int m = 0; m < NV; ++m) load_part(from, 4 * (t + m * team), d - 4 * (t + m * team), x[m]);
#pragma unroll
  for (int m = 0; m < NV; ++m) s[0] += (x[m][0] + x[m][1]) + (x[m][2] + x[m][3]);
  norm_sum<LANES>(s, red[0]);
  const float inv = 1.f / (float)d, mean = s[0] * inv;
  s[0] = 0.f;
#pragma unroll
  for (int m = 0; m < NV; ++m)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      x[m][c] = 4 * (t + m * team) + c < d ? x[m][c] - mean : 0.f;
      s[0] = fmaf(x[m][c], x[m][c], s[0]);
    }
  norm_sum<LANES>(s, red[1]);
  const float rstd = 1.f / sqrtf(fmaf(s[0], inv, k.eps));
  T* to = k.y + row * k.d;
#pragma unroll
  for (int m = 0; m < NV; ++m) {
    const uint32_t i = 4 * (t + m * team);
    const int left = d - (int)i;
    float w[4], b[4];
    if (k.w) load_part(k.w, i, left, w);
    if (k.b) load_part(k.b, i, left, b);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float h = x[m][c] * rstd;
      x[m][c] = fmaf(h, k.w ? w[c] : 1.f, k.b ? b[c] : 0.f);
    }
    store_part<STREAM>(to, i, left, x[m]);
  }
  if (k.stats && t == 0) {
    k.stats[2 * row] = mean;
    k.stats[2 * row + 1] = rstd;
  }
}

// Teams walk rows (their number, + teams, ..), the next row's loads in flight, and keep the weights' sums
// in registers.
template <typename T, int NV, int LANES>
__global__ __launch_bounds__(LANES ? 256 : 512) void layer_norm_bwd_kernel(LayerNormArgs<T> k) {
  constexpr int TEAMS = kNormTeams<LANES>;
  __shared__ float red[2][LANES ? 1 : 32];
  __shared__ float fold[TEAMS > 1 ? TEAMS - 1 : 1][TEAMS > 1 ? 4 * NV : 1][LANES ? LANES : 1];
  const int team = LANES ? LANES : blockDim.x, t = LANES ? threadIdx.x % team : threadIdx.x;
  const int number = LANES ? threadIdx.x / team : 0, d = (int)k.d;
  const float inv = 1.f / (float)d;
  float w[NV][4], sum[2][NV][4] = {};
#pragma unroll
  for (int m = 0; m < NV; ++m) {
    if (k.w) load_part(k.w, 4 * (t + m * team), d - 4 * (t + m * team), w[m]);
#pragma unroll
    for (int c = 0; c < 4; ++c) w[m][c] = k.w ? w[m][c] : 1.f;
  }
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  Quad<T> raw[2][NV];
  float mean = 0.f, rstd = 0.f;
  const auto fetch = [&](int64_t row) {
    if (row >= k.rows) return;
    mean = k.stats[2 * row], rstd = k.stats[2 * row + 1];
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const uint32_t i = 4 * (t + m * team);
      raw[0][m] = load_quad(k.x + row * k.x_row, i, d - (int)i);
      raw[1][m] = load_quad(k.dy + row * k.d, i, d - (int)i);
    }
  };
  int64_t row = (int64_t)blockIdx.x * TEAMS + number;
  int flip = 0;  // two sets of sums: one barrier a row is enough
  fetch(row);
  for (; row < k.rows; row += step, flip ^= 1) {
    float h[NV][4], g[NV][4], s[2] = {0.f, 0.f};
    const float r = rstd;
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      unpack_quad<T>(raw[0][m], h[m]);
      unpack_quad<T>(raw[1][m], g[m]);
#pragma unroll
      for (int c = 0; c < 4; ++c) h[m][c] = 4 * (t + m * team) + c < d ? (h[m][c] - mean) * r : 0.f;
    }
    fetch(row + step);
#pragma unroll
    for (int m = 0; m < NV; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        sum[0][m][c] = fmaf(g[m][c], h[m][c], sum[0][m][c]);
        sum[1][m][c] += g[m][c];
        g[m][c] *= w[m][c];
        s[0] += g[m][c];
        s[1] = fmaf(g[m][c], h[m][c], s[1]);
      }
    norm_sum<LANES>(s, red[flip]);
    s[0] *= inv, s[1] *= inv;
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const uint32_t i = 4 * (t + m * team);
#pragma unroll
      for (int c = 0; c < 4; ++c) g[m][c] = r * (g[m][c] - fmaf(h[m][c], s[1], s[0]));
      store_part(k.dx + row * k.d, i, d - (int)i, g[m]);
    }
  }
  if (!k.part) return;
  // The teams' sums, in their order.
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if constexpr (TEAMS > 1) {
      __syncthreads();
      if (number > 0) {
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
          for (int c = 0; c < 4; ++c) fold[number - 1][4 * m + c][t] = sum[j][m][c];
      }
      __syncthreads();
      if (number > 0) continue;
#pragma unroll
      for (int m = 0; m < NV; ++m)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int n = 0; n < TEAMS - 1; ++n) sum[j][m][c] += fold[n][4 * m + c][t];
    }
    float* to = k.part + ((int64_t)j * gridDim.x + blockIdx.x) * k.d;
#pragma unroll
    for (int m = 0; m < NV; ++m) store_part(to, 4 * (t + m * team), d - 4 * (t + m * team), sum[j][m]);
  }
}

// By width: teams of 16 lanes up to 64 elements, 32 up to 128, a wave up to 1024 (in steps of 256), the
// workgroup's waves beyond (16 elements a lane).
#define MQC_LN_BY_WIDTH(F)          \
  if (k.d <= 64) F(1, 16)           \
  else if (k.d <= 128) F(1, 32)     \
  else if (k.d <= 256) F(1, 64)     \
  else if (k.d <= 512) F(2, 64)     \
  else if (k.d <= 768) F(3, 64)     \
  else if (k.d <= 1024) F(4, 64)    \
  else F(4, 0)

inline int64_t layer_norm_teams(int64_t d) { return d <= 64 ? 16 : d <= 128 ? 8 : d <= 1024 ? 4 : 1; }
inline int64_t layer_norm_threads(int64_t d) { return d <= 1024 ? 256 : (d + 1023) / 1024 * 64; }

template <typename T, bool STREAM>
int launch_layer_norm_rows(const LayerNormArgs<T>& k, hipStream_t s) {
  const int64_t teams = layer_norm_teams(k.d);
  const dim3 grid((unsigned)((k.rows + teams - 1) / teams)), threads((unsigned)layer_norm_threads(k.d));
#define MQC_LN(NV, LANES) layer_norm_fwd_kernel<T, NV, LANES, STREAM><<<grid, threads, 0, s>>>(k);
  MQC_LN_BY_WIDTH(MQC_LN)
#undef MQC_LN
  return launch_status();
}
// Past the 256 MiB of the last cache y is streamed, as the gate's norms are (gate_norm.hip).
template <typename T>
int launch_layer_norm_fwd(const LayerNormArgs<T>& k, hipStream_t s) {
  return 2 * k.rows * k.d * (int64_t)sizeof(T) > (256LL << 20) ? launch_layer_norm_rows<T, true>(k, s)
                                                               : launch_layer_norm_rows<T, false>(k, s);
}

// Workgroups of the backward: each writes its sums, so not more than the card holds at once.
inline int64_t layer_norm_bwd_blocks(int64_t rows, int64_t d) {
  const int64_t teams = layer_norm_teams(d), need = (rows + teams - 1) / teams;
  const int64_t most = d <= 1024 ? 512 : 256 * (16 / (layer_norm_threads(d) / 64)) / 2;
  const int64_t each = (need + most - 1) / most;
  return (need + each - 1) / each;
}

template <typename T>
int launch_layer_norm_bwd(const LayerNormArgs<T>& k, float* dw, float* db, hipStream_t s) {
  const int64_t blocks = layer_norm_bwd_blocks(k.rows, k.d);
  const dim3 grid((unsigned)blocks), threads((unsigned)layer_norm_threads(k.d));
#define MQC_LN(NV, LANES) layer_norm_bwd_kernel<T, NV, LANES><<<grid, threads, 0, s>>>(k);
  MQC_LN_BY_WIDTH(MQC_LN)
#undef MQC_LN
  const int st = launch_status();
  if (st != MQC_OK || !k.part) return st;
  return mqc_sum_rows(k.part, dw, dw ? k.d : 0, k.part + blocks * k.d, db, db ? k.d : 0, nullptr, nullptr,
                      0, blocks, s);
}

inline int layer_norm_shape(int64_t rows, int64_t d, int64_t x_row, int dtype) {
  if (rows < 0 || d < 1) return MQC_E_SHAPE;
  if (dtype != MQC_F32 && dtype != MQC_BF16 && dtype != MQC_F16) return MQC_E_DTYPE;
  if (rows > 1 && x_row < d) return MQC_E_SHAPE;
  if (d > kLayerNormMaxWidth || rows > 0x7fffffffLL) return MQC_E_LIMIT;
  return MQC_OK;
}

template <typename T>
LayerNormArgs<T> layer_norm_args(const void* x, int64_t x_row, const float* w, int64_t rows, int64_t d) {
  LayerNormArgs<T> k{};
  k.x = (const T*)x; k.x_row = x_row; k.w = w; k.rows = rows; k.d = d;
  return k;
}

}  // namespace mqc

using namespace mqc;

#define MQC_BY_DTYPE(F)                    \
  switch (dtype) {                         \
    case MQC_F32: return F(float);         \
    case MQC_BF16: return F(bf16_t);       \
    default: return F(f16_t);              \
  }

extern "C" int64_t mqc_layer_norm_max_width(void) { return kLayerNormMaxWidth; }

extern "C" int64_t mqc_layer_norm_workspace_bytes(int64_t rows, int64_t d) {
  if (rows < 1 || d < 1) return MQC_E_SHAPE;
  if (d > kLayerNormMaxWidth) return MQC_E_LIMIT;
  return layer_norm_bwd_blocks(rows, d) * 2 * d * (int64_t)sizeof(float);
}

extern "C" int mqc_layer_norm_fwd(const void* x, int64_t x_row, const float* weight, const float* bias,
                                  void* y, float* stats, int64_t rows, int64_t d, float eps, int dtype,
                                  void* stream) {
  const int st = layer_norm_shape(rows, d, x_row, dtype);
  if (st != MQC_OK) return st;
  if (rows == 0) return MQC_OK;
  const int64_t teams = layer_norm_teams(d);
  if (!launchable((rows + teams - 1) / teams, layer_norm_threads(d))) return MQC_E_LIMIT;
  if (!x || !y) return MQC_E_NULL;
#define MQC_F(T)                                                        \
  [&] {                                                                 \
    LayerNormArgs<T> k = layer_norm_args<T>(x, x_row, weight, rows, d); \
    k.b = bias; k.eps = eps; k.y = (T*)y; k.stats = stats;              \
    return launch_layer_norm_fwd<T>(k, (hipStream_t)stream);            \
  }()
  MQC_BY_DTYPE(MQC_F)
#undef MQC_F
}

extern "C" int mqc_layer_norm_bwd(const void* x, int64_t x_row, const float* weight, const float* stats,
                                  const void* dy, void* dx, float* dweight, float* dbias, int64_t rows,
                                  int64_t d, int dtype, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  const int st = layer_norm_shape(rows, d, x_row, dtype);
  if (st != MQC_OK) return st;
  if (rows < 1) return MQC_E_SHAPE;
  const bool sums = dweight || dbias;
  if (!x || !stats || !dy || !dx || (sums && !workspace)) return MQC_E_NULL;
  if (sums && workspace_bytes < mqc_layer_norm_workspace_bytes(rows, d)) return MQC_E_SPACE;
#define MQC_F(T)                                                                \
  [&] {                                                                         \
    LayerNormArgs<T> k = layer_norm_args<T>(x, x_row, weight, rows, d);         \
    k.stats = const_cast<float*>(stats); k.dy = (const T*)dy; k.dx = (T*)dx;    \
    k.part = sums ? (float*)workspace : nullptr;                                \
    return launch_layer_norm_bwd<T>(k, dweight, dbias, (hipStream_t)stream);    \
  }()
  MQC_BY_DTYPE(MQC_F)
#undef MQC_F
}
