// The gated scan, a linear recurrence with a real state for each channel:
//   D_t = softplus(dt_t),  p_t = D_t exp(log_rate),  a_t = exp(-p_t),  s_t = sigmoid(g_t) x_t
//   h_t = a_t h_{t-1} + (1 - a_t) s_t
// (the zero-order hold of dh/dt = rate (s - h): unit gain at rest for every rate and step), where
// a reset at t takes h_{t-1} as 0. Backward, with G_t = dy_t + a_{t+1} G_{t+1} (nothing from behind a
// reset at t + 1; dh_last joins at the last step):
//   ds_t = (1 - a_t) G_t           dx_t = ds_t sigmoid(g_t)    dg_t = ds_t s_t (1 - sigmoid(g_t))
//   dp_t = a_t G_t (s_t - h_{t-1}) ddt_t = dp_t exp(log_rate) sigmoid(dt_t)
//   dlog_rate = sum over b, t of dp_t p_t,  dh0 = a_0 G_0
// States, sums and gates are fp32; y and the gradients are rounded to the storage type once.
#include "common.hpp"

namespace mqc {

// Steps of a chunk, which is walked from zero: y_t = u_t + d_t, u the chunk's own part and d what is
// left of the state before it, and the state goes from chunk to chunk by the chunk's whole decay and
// its last u. A state that grows slowly over many tokens is so rounded once a chunk, not once a
// token. A training forward stores the states between chunks.
constexpr int kScanChunk = 128;

// log(1 + e) by its series below 3/32 (the first left-out term is under 2^-24 of the sum there),
// where rounding 1 + e would lose digits.
__device__ inline float scan_softplus(float v) {
  const float e = __expf(-fabsf(v));
  const float series =
      e * (1.f - e * (0.5f - e * (1.f / 3 - e * (0.25f - e * (0.2f - e * (1.f / 6 - e * (1.f / 7)))))));
  return fmaxf(v, 0.f) + (e < 0.09375f ? series : __logf(1.f + e));
}

// A step's decay as one number c. A slow channel has a near 1 and forgets by 1 - a a token: rounding
// a to fp32 would shift its rate, and with it the gain at rest, by 2^-25 / (1 - a). So c is 1 - a
// (from its own series) while that is under a half, and -a after that; the sign bit tells.
struct ScanRate { float log_rate, rate; };
__device__ inline ScanRate scan_rate(float log_rate) { return {log_rate, expf(log_rate)}; }
__device__ inline float scan_decay(float dt, ScanRate r, float& p) {
  p = scan_softplus(dt) * r.rate;
  if (__builtin_expect(dt < -80.f, 0)) p = __expf(dt + r.log_rate);  // exp(dt) alone underflows
  p = p > 3e38f ? 3e38f : p;  // p a stays 0 there, not inf * 0; a NaN stays one
  const float a = __expf(-p);
  const float series =
      p * (1.f - p * (0.5f - p * (1.f / 6 - p * (1.f / 24 - p * (1.f / 120 - p * (1.f / 720))))));
  const float w = p < 0.25f ? series : 1.f - a;
  return w < 0.5f ? w : -a;
}
__device__ inline bool scan_fast(float c) { return __float_as_int(c) < 0; }  // c is -a
__device__ inline float scan_a(float c) { return scan_fast(c) ? -c : 1.f - c; }
__device__ inline float scan_w(float c) { return scan_fast(c) ? 1.f + c : c; }
// a v, and a h + (1 - a) s.
__device__ inline float scan_fade(float c, float v) { return scan_fast(c) ? -c * v : fmaf(-c, v, v); }
// The decay of two steps: 1 - a from its own sum, a from its own product.
struct ScanSpan {
  float a = 1.f, w = 0.f;
  __device__ void then(float c) {
    a *= scan_a(c);
    w = fmaf(scan_w(c), 1.f - w, w);
  }
  __device__ void cut() { a = 0.f, w = 1.f; }
  __device__ float c() const { return w < 0.5f ? w : -a; }
};
__device__ inline float scan_step(float c, float s, float h) {
  return fmaf(c, s - h, scan_fast(c) ? s : h);
}
template <typename T>
struct ScanArgs {
  const T *dt, *g, *x;
  int64_t dt_row, g_row, x_row;  // elements between tokens
  const float* log_rate;
  const float* h0;
  const uint8_t* reset;
  float* carries;
  int64_t seq, width;
  // forward
  T* y;
  float* h_last;
  // backward
  const T* dy;
  const float* dh_last;
  T *ddt, *dg, *dx;
  float *drate, *dh0;
};

// A lane walks one channel of one sequence.
template <typename T>
__global__ __launch_bounds__(64) void gated_scan_fwd_kernel(ScanArgs<T> k) {
  const int64_t d = (int64_t)blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (d >= k.width) return;
  const ScanRate rate = scan_rate(k.log_rate[d]);
  float h = k.h0 ? k.h0[b * k.width + d] : 0.f, u = 0.f, left = h;
  const int64_t chunks = (k.seq + kScanChunk - 1) / kScanChunk;
  ScanSpan span;
  bool cut = false;
  for (int64_t t = 0; t < k.seq; ++t) {
    const int64_t row = b * k.seq + t;
    if (t % kScanChunk == 0) {
      if (t > 0) h = cut ? u : u + scan_fade(span.c(), h);
      if (k.carries) k.carries[(b * chunks + t / kScanChunk) * k.width + d] = h;
      u = 0.f, left = h, span = ScanSpan(), cut = false;
    }
    float p, sg, cg;
    const float c = scan_decay(load_scalar(k.dt + row * k.dt_row + d), rate, p);
    sigmoid_pair(load_scalar(k.g + row * k.g_row + d), sg, cg);
    if (k.reset && k.reset[row]) u = left = 0.f, span.cut(), cut = true;
    u = scan_step(c, sg * load_scalar(k.x + row * k.x_row + d), u);
    left = scan_fade(c, left);
    span.then(c);
    store_scalar(k.y + row * k.width + d, u + left);
  }
  if (k.seq > 0) h = cut ? u : u + scan_fade(span.c(), h);
  if (k.h_last) k.h_last[b * k.width + d] = h;
}

// Backward: the chunks from the last to the first, each walked forward from its stored entry state
// with its states kept in LDS, then back.
template <typename T>
__global__ __launch_bounds__(64) void gated_scan_bwd_kernel(ScanArgs<T> k) {
  __shared__ float states[kScanChunk][64];
  const int64_t d = (int64_t)blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (d >= k.width) return;
  const int64_t chunks = (k.seq + kScanChunk - 1) / kScanChunk;
  const ScanRate rate = scan_rate(k.log_rate[d]);
  float G = k.dh_last ? k.dh_last[b * k.width + d] : 0.f, drate = 0.f;
  for (int64_t j = chunks - 1; j >= 0; --j) {
    const int64_t t0 = j * kScanChunk;
    const int n = (int)(k.seq - t0 < kScanChunk ? k.seq - t0 : kScanChunk);
    float left = k.carries[(b * chunks + j) * k.width + d], u = 0.f;
    for (int i = 0; i < n; ++i) {
      const int64_t row = b * k.seq + t0 + i;
      float p, sg, cg;
      const float c = scan_decay(load_scalar(k.dt + row * k.dt_row + d), rate, p);
      sigmoid_pair(load_scalar(k.g + row * k.g_row + d), sg, cg);
      if (k.reset && k.reset[row]) u = left = 0.f;
      states[i][threadIdx.x] = u + left;
      u = scan_step(c, sg * load_scalar(k.x + row * k.x_row + d), u);
      left = scan_fade(c, left);
    }
    for (int i = n - 1; i >= 0; --i) {
      const int64_t row = b * k.seq + t0 + i;
      const float dtv = load_scalar(k.dt + row * k.dt_row + d);
      float p, sg, cg, sd, cd;
      const float c = scan_decay(dtv, rate, p);
      sigmoid_pair(load_scalar(k.g + row * k.g_row + d), sg, cg);
      sigmoid_pair(dtv, sd, cd);
      const float s = sg * load_scalar(k.x + row * k.x_row + d);
      G += load_scalar(k.dy + row * k.width + d);
      const float dp = scan_a(c) * G * (s - states[i][threadIdx.x]);
      const float ds = scan_w(c) * G;
      store_scalar(k.ddt + row * k.width + d, dp * rate.rate * sd);
      store_scalar(k.dg + row * k.width + d, ds * s * cg);
      store_scalar(k.dx + row * k.width + d, ds * sg);
      drate = fmaf(dp, p, drate);
      G = k.reset && k.reset[row] ? 0.f : scan_fade(c, G);
    }
  }
  k.drate[b * k.width + d] = drate;
  if (k.dh0) k.dh0[b * k.width + d] = G;
}

// One token for each sequence, the state in place.
template <typename T>
__global__ __launch_bounds__(256) void gated_scan_step_kernel(ScanArgs<T> k, float* h) {
  const int64_t d = (int64_t)blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
  if (d >= k.width) return;
  float p, sg, cg;
  const float c = scan_decay(load_scalar(k.dt + b * k.dt_row + d), scan_rate(k.log_rate[d]), p);
  sigmoid_pair(load_scalar(k.g + b * k.g_row + d), sg, cg);
  const float v = scan_step(c, sg * load_scalar(k.x + b * k.x_row + d), h[b * k.width + d]);
  h[b * k.width + d] = v;
  store_scalar(k.y + b * k.width + d, v);
}

template <typename T>
int launch_gated_scan_fwd(const ScanArgs<T>& k, int64_t batch, hipStream_t s) {
  gated_scan_fwd_kernel<T><<<dim3((unsigned)((k.width + 63) / 64), (unsigned)batch), dim3(64), 0, s>>>(k);
  return launch_status();
}

template <typename T>
int launch_gated_scan_bwd(ScanArgs<T> k, int64_t batch, float* drate, hipStream_t s) {
  gated_scan_bwd_kernel<T><<<dim3((unsigned)((k.width + 63) / 64), (unsigned)batch), dim3(64), 0, s>>>(k);
  const int st = launch_status();
  if (st != MQC_OK) return st;
  return mqc_sum_rows(k.drate, drate, k.width, nullptr, nullptr, 0, nullptr, nullptr, 0, batch, s);
}

template <typename T>
int launch_gated_scan_step(const ScanArgs<T>& k, float* h, int64_t batch, hipStream_t s) {
  gated_scan_step_kernel<T>
      <<<dim3((unsigned)((k.width + 255) / 256), (unsigned)batch), dim3(256), 0, s>>>(k, h);
  return launch_status();
}

// The sizes that every entry point takes: rows hold `width` elements, grids fit.
inline int scan_shape(int64_t batch, int64_t seq, int64_t width, int64_t dt_row, int64_t g_row,
                      int64_t x_row, int dtype) {
  if (batch < 0 || seq < 0 || width < 0) return MQC_E_SHAPE;
  if (dtype != MQC_F32 && dtype != MQC_BF16 && dtype != MQC_F16) return MQC_E_DTYPE;
  if (batch * seq > 1 && (dt_row < width || g_row < width || x_row < width)) return MQC_E_SHAPE;
  if (batch > 65535 || seq > (1LL << 31) || width > (1LL << 31)) return MQC_E_LIMIT;
  return MQC_OK;
}

template <typename T>
ScanArgs<T> scan_args(const void* dt, int64_t dt_row, const void* g, int64_t g_row, const void* x,
                      int64_t x_row, const float* log_rate, const void* reset, int64_t seq,
                      int64_t width) {
  ScanArgs<T> k{};
  k.dt = (const T*)dt; k.g = (const T*)g; k.x = (const T*)x;
  k.dt_row = dt_row; k.g_row = g_row; k.x_row = x_row;
  k.log_rate = log_rate; k.reset = (const uint8_t*)reset;
  k.seq = seq; k.width = width;
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

extern "C" int mqc_gated_scan_chunk(void) { return kScanChunk; }

extern "C" int64_t mqc_gated_scan_workspace_bytes(int64_t batch, int64_t seq_len, int64_t width) {
  if (batch < 0 || seq_len < 0 || width < 0) return MQC_E_SHAPE;
  return batch * width * (int64_t)sizeof(float);
}

extern "C" int mqc_gated_scan_fwd(const void* dt, int64_t dt_row, const void* g, int64_t g_row,
                                  const void* x, int64_t x_row, const float* log_rate,
                                  const float* h0, const void* reset, void* y, float* h_last,
                                  float* carries, int64_t batch, int64_t seq_len, int64_t width,
                                  int dtype, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  const int st = scan_shape(batch, seq_len, width, dt_row, g_row, x_row, dtype);
  if (st != MQC_OK) return st;
  if (batch == 0 || width == 0) return MQC_OK;
  if (!log_rate || (seq_len > 0 && (!dt || !g || !x || !y))) return MQC_E_NULL;
  if (seq_len == 0 && !h_last) return MQC_OK;
  if (workspace_bytes < mqc_gated_scan_workspace_bytes(batch, seq_len, width)) return MQC_E_SPACE;
  if (workspace_bytes > 0 && !workspace) return MQC_E_NULL;
#define MQC_F(T)                                                                               \
  [&] {                                                                                        \
    ScanArgs<T> k = scan_args<T>(dt, dt_row, g, g_row, x, x_row, log_rate, reset, seq_len, width); \
    k.h0 = h0; k.y = (T*)y; k.h_last = h_last; k.carries = carries;                            \
    return launch_gated_scan_fwd<T>(k, batch, (hipStream_t)stream);                            \
  }()
  MQC_BY_DTYPE(MQC_F)
#undef MQC_F
}

extern "C" int mqc_gated_scan_bwd(const void* dt, int64_t dt_row, const void* g, int64_t g_row,
                                  const void* x, int64_t x_row, const float* log_rate,
                                  const void* reset, const float* carries, const void* dy,
                                  const float* dh_last, void* ddt, void* dg, void* dx,
                                  float* dlog_rate, float* dh0, int64_t batch, int64_t seq_len,
                                  int64_t width, int dtype, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const int st = scan_shape(batch, seq_len, width, dt_row, g_row, x_row, dtype);
  if (st != MQC_OK) return st;
  if (batch < 1 || seq_len < 1 || width < 1) return MQC_E_SHAPE;
  if (!dt || !g || !x || !log_rate || !carries || !dy || !ddt || !dg || !dx || !dlog_rate ||
      !workspace)
    return MQC_E_NULL;
  if (workspace_bytes < mqc_gated_scan_workspace_bytes(batch, seq_len, width)) return MQC_E_SPACE;
#define MQC_F(T)                                                                               \
  [&] {                                                                                        \
    ScanArgs<T> k = scan_args<T>(dt, dt_row, g, g_row, x, x_row, log_rate, reset, seq_len, width); \
    k.carries = const_cast<float*>(carries);                                                   \
    k.dy = (const T*)dy; k.dh_last = dh_last; k.ddt = (T*)ddt; k.dg = (T*)dg; k.dx = (T*)dx;    \
    k.drate = (float*)workspace; k.dh0 = dh0;                                                  \
    return launch_gated_scan_bwd<T>(k, batch, dlog_rate, (hipStream_t)stream);                 \
  }()
  MQC_BY_DTYPE(MQC_F)
#undef MQC_F
}

extern "C" int mqc_gated_scan_step(const void* dt, int64_t dt_row, const void* g, int64_t g_row,
                                   const void* x, int64_t x_row, const float* log_rate, float* h,
                                   void* y, int64_t batch, int64_t width, int dtype,
                                   void* stream) {
  const int st = scan_shape(batch, 1, width, dt_row, g_row, x_row, dtype);
  if (st != MQC_OK) return st;
  if (batch == 0 || width == 0) return MQC_OK;
  if (!dt || !g || !x || !log_rate || !h || !y) return MQC_E_NULL;
#define MQC_F(T)                                                                               \
  [&] {                                                                                        \
    ScanArgs<T> k = scan_args<T>(dt, dt_row, g, g_row, x, x_row, log_rate, nullptr, 1, width);  \
    k.y = (T*)y;                                                                               \
    return launch_gated_scan_step<T>(k, h, batch, (hipStream_t)stream);                        \
  }()
  MQC_BY_DTYPE(MQC_F)
#undef MQC_F
}
