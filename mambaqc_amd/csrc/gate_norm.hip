// What stands between two blocks of a pre-norm and post-norm stack, in one pass over the row:
//   v = sigmoid(z) y,  rho = 1 / sqrt(mean v^2 + eps),  r = v rho post
//   o = x + scale r,   tau = 1 / sqrt(mean o^2 + eps),  n = o tau pre
// o is the residual stream, n what the next block reads; without z the gate is 1, without post r = v.
// Backward, from do and dn (means over the row, w = scale post, u = dn pre):
//   O = do + tau u - o tau^3 mean(u o)                                (the gradient of o, dx = O)
//   dv = rho w O - v rho^3 mean(w O v)   (without post dv = scale O)  dy = dv sigmoid(z)
//   dz = dv v (1 - sigmoid(z)),  dscale = sum over rows of O r,  dpost = sum of scale O v rho,
//   dpre = sum of dn o tau
// mean(w O v) splits into mean(w v (do + tau u)) - tau^3 mean(u o) mean(w v o), so that a row takes
// one reduction (of three sums) and not two, the second waiting for the first.
// Everything between the loads and the stores is fp32; n comes from o before o is rounded.
//
// A row stays in registers between its loads and stores, so memory bounds both directions. bf16, 8192 x
// 768: forward 14.4 us (63 MB, 4.4 TB/s), backward 21 us and 5 for the weights' sums (101 MB, 4.8 TB/s;
// without the next row's loads ahead 44); 32768 x 1024 in fp16 51 us (6.5 TB/s, its inputs partly in the
// last cache; 71 when they are not), in fp32 144 and 195 (671 and 1074 MB, 4.7 and 5.5 TB/s); 65536 x 64 10 and 19 (a wave to a row instead of 16 lanes: 28 and 56).
#include "common.hpp"

namespace mqc {

template <typename T>
struct GateNormArgs {
  const T *x, *y, *z;
  int64_t z_row;  // elements between rows of z
  const float *post, *scale, *pre;
  int64_t rows, d;
  float eps;
  // forward
  T *out, *n;
  float* stats;  // [rows, 2]: rho and tau, or NULL
  // backward
  const T *dout, *dn;
  T *dx, *dy, *dz;
  float* part;  // [3, workgroups, d]: sums of O r, dn o tau, and scale O v rho
};

// Four consecutive elements from wherever they start (rows of odd widths do not start at multiples
// of a vector; gfx950 loads and stores those as it does aligned ones), `left` of them, as they are
// in memory.
template <typename T>
using Quad = uint32_t __attribute__((ext_vector_type(sizeof(T)), aligned(sizeof(T))));
template <typename T>
__device__ inline Quad<T> load_quad(const T* row, uint32_t i, int left) {
  const T* p = row + i;
  if (left >= 4) return *reinterpret_cast<const Quad<T>*>(p);
  Quad<T> v = {};
#pragma unroll
  for (int c = 0; c < 3; ++c)
    if (c < left) {
      if constexpr (sizeof(T) == 4) v[c] = __builtin_bit_cast(uint32_t, p[c]);
      else v[c / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[c]) << (16 * (c % 2));
    }
  return v;
}
template <typename T>
__device__ inline void unpack_quad(Quad<T> v, float (&out)[4]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if constexpr (sizeof(T) == 4) out[c] = __uint_as_float(v[c]);
    else out[c] = io<T>::bits_to_f32(c & 1 ? v[c / 2] >> 16 : v[c / 2] & 0xffffu);
  }
}
template <typename T>
__device__ inline void load_part(const T* row, uint32_t i, int left, float (&out)[4]) {
  unpack_quad<T>(load_quad(row, i, left), out);
}
template <bool STREAM = false, typename T>
__device__ inline void store_part(T* row, uint32_t i, int left, const float (&in)[4]) {
  T* p = row + i;
  if (left >= 4) {
    Quad<T> v;
#pragma unroll
    for (int c = 0; c < (int)sizeof(T); ++c)
      if constexpr (sizeof(T) == 4) v[c] = __float_as_uint(in[c]);
      else v[c] = pack2<T>(in[2 * c], in[2 * c + 1]);
    if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<Quad<T>*>(p));
    else *reinterpret_cast<Quad<T>*>(p) = v;
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c < left) store_scalar(p + c, in[c]);
  }
}

// A row belongs to a team of LANES lanes: 16 or 32 for narrow rows (which would leave most of a wave
// idle), a wave, or all waves of the workgroup (LANES 0). Its sums, the same in every lane; `red` holds
// 16 floats a sum.
template <int LANES, int N>
__device__ inline void team_sum(float (&v)[N], float* red) {
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
    for (int i = 0; i < N; ++i) v[i] = 0.f;
#pragma unroll 2
    for (int w = 0; w < waves; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += red[16 * i + w];
    }
  }
}

// Teams of a workgroup, and a team's number in it (uniform over a wave where that is one team's).
template <int LANES>
constexpr int kTeams = LANES ? 256 / LANES : 1;
template <int LANES>
__device__ inline int team_number() {
  if constexpr (LANES == 0) return 0;
  const int i = threadIdx.x / (LANES ? LANES : 1);
  return LANES == 64 ? __builtin_amdgcn_readfirstlane(i) : i;
}

// A lane holds elements 4 (lane + team m) + 0..3 of its row for m < NV.
template <typename T, int NV, int LANES, bool STREAM>
__global__ __launch_bounds__(LANES ? 256 : 1024) void gate_norm_fwd_kernel(GateNormArgs<T> k) {
  __shared__ float red[LANES ? 1 : 32];
  const int team = LANES ? LANES : blockDim.x, t = LANES ? threadIdx.x % team : threadIdx.x;
  const int d = (int)k.d;
  const int64_t row = (int64_t)blockIdx.x * kTeams<LANES> + team_number<LANES>();
  if (row >= k.rows) return;  // whole teams; a team of several waves has its row
  const int64_t base = row * k.d;
  float x[NV][4], v[NV][4];
  float s[1] = {0.f};
#pragma unroll
  for (int m = 0; m < NV; ++m) {
    const uint32_t i = 4 * (t + m * team);
    const int left = d - (int)i;
    load_part(k.x + base, i, left, x[m]);
    load_part(k.y + base, i, left, v[m]);
    if (k.z) {
      float z[4];
      load_part(k.z + row * k.z_row, i, left, z);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float sg, cg;
        sigmoid_pair(z[c], sg, cg);
        v[m][c] *= sg;
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) s[0] = fmaf(v[m][c], v[m][c], s[0]);
  }
  const float inv = 1.f / (float)k.d;
  float rho = 1.f;
  if (k.post) {
    team_sum<LANES>(s, red);
    rho = 1.f / sqrtf(s[0] * inv + k.eps);
  }
  s[0] = 0.f;
#pragma unroll
  for (int m = 0; m < NV; ++m) {
    const uint32_t i = 4 * (t + m * team);
    const int left = d - (int)i;
    float sc[4], po[4];
    load_part(k.scale, i, left, sc);
    if (k.post) load_part(k.post, i, left, po);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float r = k.post ? v[m][c] * rho * po[c] : v[m][c];
      x[m][c] = fmaf(sc[c], r, x[m][c]);
      s[0] = fmaf(x[m][c], x[m][c], s[0]);
    }
    store_part<STREAM>(k.out + base, i, left, x[m]);
  }
  team_sum<LANES>(s, red + (LANES ? 0 : 16));
  const float tau = 1.f / sqrtf(s[0] * inv + k.eps);
#pragma unroll
  for (int m = 0; m < NV; ++m) {
    const uint32_t i = 4 * (t + m * team);
    const int left = d - (int)i;
    float pre[4];
    load_part(k.pre, i, left, pre);
#pragma unroll
    for (int c = 0; c < 4; ++c) x[m][c] *= tau * pre[c];
    store_part<STREAM>(k.n + base, i, left, x[m]);
  }
  if (k.stats && t == 0) {
    k.stats[2 * row] = rho;
    k.stats[2 * row + 1] = tau;
  }
}

// Teams walk rows (their number, + teams, ..) and keep the weights' sums in registers.
template <typename T, int NV, int LANES>
__global__ __launch_bounds__(LANES ? 256 : 1024) void gate_norm_bwd_kernel(GateNormArgs<T> k) {
  __shared__ float red[2][LANES ? 1 : 48];
  __shared__ float fold[LANES ? kTeams<LANES> - 1 : 1][LANES ? 12 * NV : 1][LANES ? LANES : 1];
  // The weights' sums: in registers, or where 1024 threads have too few, in LDS.
  constexpr bool IN_LDS = NV > 1;
  __shared__ float held[IN_LDS ? 3 * NV * 4 : 1][IN_LDS ? 1024 : 1];
  const int team = LANES ? LANES : blockDim.x, t = LANES ? threadIdx.x % team : threadIdx.x;
  const int number = team_number<LANES>(), d = (int)k.d;
  const float inv = 1.f / (float)k.d;
  float sum[3][IN_LDS ? 1 : NV][4], sc[NV][4], po[NV][4], pre[NV][4];
  const auto weights = [&] {
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const uint32_t i = 4 * (t + m * team);
      const int left = d - (int)i;
      load_part(k.scale, i, left, sc[m]);
      load_part(k.pre, i, left, pre[m]);
      if (k.post) load_part(k.post, i, left, po[m]);
#pragma unroll
      for (int c = 0; c < 4; ++c) po[m][c] = k.post ? po[m][c] : 1.f;
    }
  };
  if constexpr (NV == 1) weights();
#pragma unroll
  for (int j = 0; j < 3; ++j)
#pragma unroll
    for (int m = 0; m < NV; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (IN_LDS) held[(j * NV + m) * 4 + c][t] = 0.f;
        else sum[j][m][c] = 0.f;
      }
  const auto add = [&](int j, int m, int c, float a, float b) {
    if constexpr (IN_LDS) {
      float& at = held[(j * NV + m) * 4 + c][t];
      at = fmaf(a, b, at);
    } else {
      sum[j][m][c] = fmaf(a, b, sum[j][m][c]);
    }
  };
  const int64_t first = (int64_t)blockIdx.x * kTeams<LANES> + number;
  const int64_t step = (int64_t)gridDim.x * kTeams<LANES>;
  int flip = 0;  // two sets of sums: one barrier a row is enough
  // A row's loads go out while the row before is worked on (workgroups are few: each writes its sums),
  // where the registers are there for it.
  constexpr bool AHEAD = NV == 1;
  Quad<T> raw[5][AHEAD ? NV : 1];
  float rho = 1.f, tau = 1.f;
  const auto fetch = [&](int64_t row, int m, int to) {
    const int64_t base = row * k.d;
    const uint32_t i = 4 * (t + m * team);
    const int left = d - (int)i;
    raw[0][to] = load_quad(k.x + base, i, left);
    raw[1][to] = load_quad(k.y + base, i, left);
    if (k.z) raw[2][to] = load_quad(k.z + row * k.z_row, i, left);
    if (k.dout) raw[3][to] = load_quad(k.dout + base, i, left);
    if (k.dn) raw[4][to] = load_quad(k.dn + base, i, left);
  };
  const auto ahead = [&](int64_t row) {
    if (!AHEAD || row >= k.rows) return;
    rho = k.stats[2 * row], tau = k.stats[2 * row + 1];
#pragma unroll
    for (int m = 0; m < NV; ++m) fetch(row, m, AHEAD ? m : 0);
  };
  ahead(first);
  for (int64_t row = first; row < k.rows; row += step, flip ^= 1) {
    const int64_t base = row * k.d;
    const float rho_now = AHEAD ? rho : k.stats[2 * row], tau_now = AHEAD ? tau : k.stats[2 * row + 1];
    float o[NV][4], v[NV][4], sg[NV][4], cg[NV][4], dn[NV][4], g[NV][4];
    float s[3] = {0.f, 0.f, 0.f};
    if constexpr (NV > 1) weights();
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const int at = AHEAD ? m : 0;
      if (!AHEAD) fetch(row, m, at);
      unpack_quad<T>(raw[0][at], o[m]);
      unpack_quad<T>(raw[1][at], v[m]);
      if (k.z) unpack_quad<T>(raw[2][at], sg[m]);
      if (k.dout) unpack_quad<T>(raw[3][at], g[m]);
      if (k.dn) unpack_quad<T>(raw[4][at], dn[m]);
    }
    ahead(row + step);
#pragma unroll
    for (int m = 0; m < NV; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (!k.dout) g[m][c] = 0.f;
        if (!k.dn) dn[m][c] = 0.f;
        if (k.z) {
          sigmoid_pair(sg[m][c], sg[m][c], cg[m][c]);
          v[m][c] *= sg[m][c];
        }
        o[m][c] = fmaf(sc[m][c], v[m][c] * rho_now * po[m][c], o[m][c]);
        const float u = dn[m][c] * pre[m][c], wv = sc[m][c] * po[m][c] * v[m][c];
        g[m][c] = fmaf(tau_now, u, g[m][c]);
        add(1, m, c, dn[m][c] * tau_now, o[m][c]);
        s[0] = fmaf(u, o[m][c], s[0]);
        s[1] = fmaf(wv, g[m][c], s[1]);
        s[2] = fmaf(wv, o[m][c], s[2]);
      }
    team_sum<LANES>(s, red[flip]);
    if constexpr (NV > 1) weights();  // not held meanwhile, nor z's gates: a lane has 128 registers
    // Of rows near zero under a small eps, a norm's cube alone would be infinite.
    const auto cubed = [](float norm, float v) { return norm * (norm * (norm * v)); };
    const float back = cubed(tau_now, s[0] * inv);
    const float side = k.post ? cubed(rho_now, (s[1] - back * s[2]) * inv) : 0.f;
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const uint32_t i = 4 * (t + m * team);
      const int left = d - (int)i;
      float dy[4], dz[4];
      if constexpr (NV > 1) {
        if (k.z) {
          load_part(k.z + row * k.z_row, i, left, sg[m]);
#pragma unroll
          for (int c = 0; c < 4; ++c) sigmoid_pair(sg[m][c], sg[m][c], cg[m][c]);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float O = fmaf(-back, o[m][c], g[m][c]), vr = v[m][c] * rho_now;
        add(0, m, c, O, vr * po[m][c]);
        add(2, m, c, sc[m][c] * O, vr);
        g[m][c] = O;
        const float dv = fmaf(rho_now * sc[m][c] * po[m][c], O, -side * v[m][c]);
        dy[c] = k.z ? dv * sg[m][c] : dv;
        dz[c] = k.z ? dv * v[m][c] * cg[m][c] : 0.f;
      }
      store_part(k.dx + base, i, left, g[m]);
      store_part(k.dy + base, i, left, dy);
      if (k.z) store_part(k.dz + base, i, left, dz);
    }
  }
  if constexpr (LANES > 0) {  // the workgroup's teams into its first, in order
    if (number > 0) {
#pragma unroll
      for (int j = 0; j < 3; ++j)
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
          for (int c = 0; c < 4; ++c) fold[number - 1][(j * NV + m) * 4 + c][t] = sum[j][m][c];
    }
    __syncthreads();
    if (number > 0) return;
#pragma unroll 1
    for (int w = 0; w < kTeams<LANES> - 1; ++w)
#pragma unroll
      for (int j = 0; j < 3; ++j)
#pragma unroll
        for (int m = 0; m < NV; ++m)
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[j][m][c] += fold[w][(j * NV + m) * 4 + c][t];
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
#pragma unroll
    for (int m = 0; m < NV; ++m) {
      const uint32_t i = 4 * (t + m * team);
      if constexpr (IN_LDS) {
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[j][0][c] = held[(j * NV + m) * 4 + c][t];
      }
      store_part(k.part + ((int64_t)j * gridDim.x + blockIdx.x) * k.d, i, d - (int)i, sum[j][IN_LDS ? 0 : m]);
    }
}

constexpr int64_t kGateNormMaxWidth = 8192;

// A backward's workgroups: as many as run at once (16 waves a CU, by their registers), so that all of
// them walk about as many rows, and no more, since each writes 12 d bytes of sums.
inline int64_t gate_norm_bwd_teams(int64_t d) { return d <= 64 ? 16 : d <= 128 ? 8 : d <= 256 ? 4 : 1; }
inline int64_t gate_norm_bwd_waves(int64_t d) {
  return d <= 256 ? 4 : d <= 4096 ? (d + 255) / 256 : (d + 511) / 512;
}
inline int64_t gate_norm_bwd_blocks(int64_t rows, int64_t d) {
  const int64_t teams = gate_norm_bwd_teams(d), need = (rows + teams - 1) / teams;
  const int64_t most = 256 * (16 / gate_norm_bwd_waves(d));
  const int64_t each = (need + most - 1) / most;
  return (need + each - 1) / each;
}

// STREAM: stores that leave no copy in the caches, where x, y, z, out and n are more than the 256 MiB
// of the last of them: 32768 x 1024 in fp16 (320 MiB) 51 us against 74, 32768 x 512 30 and 31; below,
// the next product finds n in the cache.
template <typename T, bool STREAM>
int launch_gate_norm_rows(const GateNormArgs<T>& k, hipStream_t s) {
#define MQC_GN(NV, LANES)                                                                       \
  gate_norm_fwd_kernel<T, NV, LANES, STREAM>                                                    \
      <<<dim3((unsigned)((k.rows + kTeams<LANES> - 1) / kTeams<LANES>)),                        \
         dim3(LANES ? 256 : 64 * (unsigned)((k.d + 1023) / 1024)), 0, s>>>(k);                  \
  return launch_status();
  if (k.d <= 64) { MQC_GN(1, 16) }
  if (k.d <= 128) { MQC_GN(1, 32) }
  if (k.d <= 256) { MQC_GN(1, 64) }
  if (k.d <= 512) { MQC_GN(2, 64) }
  if (k.d <= 768) { MQC_GN(3, 64) }
  if (k.d <= 1024) { MQC_GN(4, 64) }
  MQC_GN(4, 0)
#undef MQC_GN
}
template <typename T>
int launch_gate_norm_fwd(const GateNormArgs<T>& k, hipStream_t s) {
  const int64_t bytes = k.rows * k.d * (int64_t)sizeof(T) * (k.z ? 5 : 4);
  return bytes > (256LL << 20) ? launch_gate_norm_rows<T, true>(k, s) : launch_gate_norm_rows<T, false>(k, s);
}

template <typename T>
int launch_gate_norm_bwd(const GateNormArgs<T>& k, float* dscale, float* dpre, float* dpost,
                         hipStream_t s) {
  const int64_t blocks = gate_norm_bwd_blocks(k.rows, k.d), waves = gate_norm_bwd_waves(k.d);
#define MQC_GN(NV, LANES) \
  gate_norm_bwd_kernel<T, NV, LANES><<<dim3((unsigned)blocks), dim3(64 * (unsigned)waves), 0, s>>>(k);
  if (k.d <= 64) { MQC_GN(1, 16) }
  else if (k.d <= 128) { MQC_GN(1, 32) }
  else if (k.d <= 256) { MQC_GN(1, 64) }
  else if (k.d <= 4096) { MQC_GN(1, 0) }
  else { MQC_GN(2, 0) }
#undef MQC_GN
  const int st = launch_status();
  if (st != MQC_OK) return st;
  const int64_t each = blocks * k.d;
  return mqc_sum_rows(k.part, dscale, k.d, k.part + each, dpre, k.d, k.part + 2 * each, dpost,
                      dpost ? k.d : 0, blocks, s);
}

inline int gate_norm_shape(int64_t rows, int64_t d, const void* z, int64_t z_row, int dtype) {
  if (rows < 0 || d < 1) return MQC_E_SHAPE;
  if (dtype != MQC_F32 && dtype != MQC_BF16 && dtype != MQC_F16) return MQC_E_DTYPE;
  if (z && rows > 1 && z_row < d) return MQC_E_SHAPE;
  if (d > kGateNormMaxWidth || rows > 0x7fffffffLL) return MQC_E_LIMIT;
  return MQC_OK;
}
// The forward's rows are bounded by their launch (launch_gate_norm_rows; the backward's workgroups walk).
inline bool gate_norm_fwd_fits(int64_t rows, int64_t d) {
  const int64_t teams = d <= 64 ? 16 : d <= 128 ? 8 : d <= 1024 ? 4 : 1;
  return launchable((rows + teams - 1) / teams, d <= 1024 ? 256 : 64 * ((d + 1023) / 1024));
}

template <typename T>
GateNormArgs<T> gate_norm_args(const void* x, const void* y, const void* z, int64_t z_row,
                               const float* post, const float* scale, const float* pre,
                               int64_t rows, int64_t d, float eps) {
  GateNormArgs<T> k{};
  k.x = (const T*)x; k.y = (const T*)y; k.z = (const T*)z; k.z_row = z_row;
  k.post = post; k.scale = scale; k.pre = pre;
  k.rows = rows; k.d = d; k.eps = eps;
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

extern "C" int64_t mqc_gate_norm_max_width(void) { return kGateNormMaxWidth; }

extern "C" int64_t mqc_gate_norm_workspace_bytes(int64_t rows, int64_t d) {
  if (rows < 1 || d < 1) return MQC_E_SHAPE;
  if (d > kGateNormMaxWidth) return MQC_E_LIMIT;
  return gate_norm_bwd_blocks(rows, d) * 3 * d * (int64_t)sizeof(float);
}

extern "C" int mqc_gate_norm_fwd(const void* x, const void* y, const void* z, int64_t z_row,
                                 const float* post, const float* scale, const float* pre, void* out,
                                 void* n, float* stats, int64_t rows, int64_t d, float eps,
                                 int dtype, void* stream) {
  const int st = gate_norm_shape(rows, d, z, z_row, dtype);
  if (st != MQC_OK) return st;
  if (rows == 0) return MQC_OK;
  if (!gate_norm_fwd_fits(rows, d)) return MQC_E_LIMIT;
  if (!x || !y || !scale || !pre || !out || !n) return MQC_E_NULL;
#define MQC_F(T)                                                                        \
  [&] {                                                                                 \
    GateNormArgs<T> k = gate_norm_args<T>(x, y, z, z_row, post, scale, pre, rows, d, eps); \
    k.out = (T*)out; k.n = (T*)n; k.stats = stats;                                      \
    return launch_gate_norm_fwd<T>(k, (hipStream_t)stream);                             \
  }()
  MQC_BY_DTYPE(MQC_F)
#undef MQC_F
}

extern "C" int mqc_gate_norm_bwd(const void* x, const void* y, const void* z, int64_t z_row,
                                 const float* post, const float* scale, const float* pre,
                                 const float* stats, const void* dout, const void* dn, void* dx,
                                 void* dy, void* dz, float* dpost, float* dscale, float* dpre,
                                 int64_t rows, int64_t d, int dtype, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  const int st = gate_norm_shape(rows, d, z, z_row, dtype);
  if (st != MQC_OK) return st;
  if (rows < 1) return MQC_E_SHAPE;
  if (!x || !y || !scale || !pre || !stats || !dx || !dy || (z && !dz) || (post && !dpost) ||
      !dscale || !dpre || !workspace)
    return MQC_E_NULL;
  if (workspace_bytes < mqc_gate_norm_workspace_bytes(rows, d)) return MQC_E_SPACE;
#define MQC_F(T)                                                                       \
  [&] {                                                                                \
    GateNormArgs<T> k = gate_norm_args<T>(x, y, z, z_row, post, scale, pre, rows, d, 0.f); \
    k.stats = const_cast<float*>(stats);                                               \
    k.dout = (const T*)dout; k.dn = (const T*)dn;                                      \
    k.dx = (T*)dx; k.dy = (T*)dy; k.dz = (T*)dz; k.part = (float*)workspace;           \
    return launch_gate_norm_bwd<T>(k, dscale, dpre, post ? dpost : nullptr, (hipStream_t)stream); \
  }()
  MQC_BY_DTYPE(MQC_F)
#undef MQC_F
}
