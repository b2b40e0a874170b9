// C ABI of the gated delta rule (kernels: gated_delta.hpp).
#include "gated_delta.hpp"

using namespace mqc;

namespace {

int64_t key_width(int64_t k_dim) { return k_dim <= 32 ? 32 : k_dim <= 64 ? 64 : 128; }
int64_t value_width(int64_t v_dim) { return (v_dim + 31) / 32 * 32; }
int64_t chunk_count(int64_t seq) { return (seq + delta::kC - 1) / delta::kC; }

// Where the workspace's parts begin, each a multiple of 256 bytes long.
struct Space {
  int64_t keys, tri, zeros, vec, dstates, z, dq, dk, bytes;
};
Space space(int64_t batch, int64_t seq, int64_t k_heads, int64_t v_heads, int64_t k_dim, int64_t v_dim,
            int dtype, bool backward) {
  const int64_t pieces = dtype == MQC_BF16 ? 1 : dtype == MQC_F16 ? 2 : 3;
  const int64_t kd = key_width(k_dim), vp = value_width(v_dim);
  const int64_t units = batch * k_heads * chunk_count(seq), parts = batch * v_heads * chunk_count(seq);
  const int64_t frag = delta::kFrag * 2;
  Space w{};
  const auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  w.keys = take(units * 3 * kd / 8 * pieces * frag);
  w.tri = take(parts * 2 * delta::kTri * delta::kPieces * frag);
  w.zeros = take(delta::kPieces * frag);
  w.vec = take(parts * 4 * delta::kC * 4);
  if (backward) {
    w.dstates = take(parts * kd * vp * 4);
    w.z = take(parts * delta::kC * vp * 4);
    if (k_heads != v_heads) {
      w.dq = take(batch * seq * v_heads * k_dim * 4);
      w.dk = take(batch * seq * v_heads * k_dim * 4);
    }
  }
  return w;
}

int shape(int64_t batch, int64_t seq, int64_t k_heads, int64_t v_heads, int64_t k_dim, int64_t v_dim,
          int dtype, int g_type, int beta_type, bool backward) {
  if (batch < 0 || seq < 0 || k_heads < 1 || v_heads < 1 || k_dim < 1 || v_dim < 1 ||
      v_heads % k_heads)
    return MQC_E_SHAPE;
  for (int d : {dtype, g_type, beta_type})
    if (d != MQC_F32 && d != MQC_BF16 && d != MQC_F16) return MQC_E_DTYPE;
  if (k_dim > delta::kMaxK || v_dim > (1 << 20) || batch > (1 << 24) || v_heads > (1 << 24) ||
      seq > (1LL << 31))
    return MQC_E_LIMIT;
  const int64_t heads = batch * v_heads;  // at most 2^48; the rest below 2^63 once this is small
  if (heads > (1 << 26) || !launchable(heads * chunk_count(seq), backward ? 1024 : 256) ||
      !launchable(heads * (value_width(v_dim) / 16), 256))
    return MQC_E_LIMIT;
  if (batch * seq > (1LL << 40) / (v_heads * k_dim)) return MQC_E_LIMIT;
  return MQC_OK;
}

template <typename T>
delta::Args<T> args(const void* q, const void* k, const void* v, const int64_t* strides, const void* g,
                    int g_type, const void* beta, int beta_type, int64_t batch, int64_t seq,
                    int64_t k_heads, int64_t v_heads, int64_t k_dim, int64_t v_dim, float scale) {
  delta::Args<T> a{};
  a.q = (const T*)q; a.k = (const T*)k; a.v = (const T*)v;
  a.q_b = strides[0]; a.q_t = strides[1]; a.q_h = strides[2];
  a.k_b = strides[3]; a.k_t = strides[4]; a.k_h = strides[5];
  a.v_b = strides[6]; a.v_t = strides[7]; a.v_h = strides[8];
  a.g = g; a.g_type = g_type; a.beta = beta; a.beta_type = beta_type;
  a.batch = batch; a.seq = seq; a.k_heads = k_heads; a.v_heads = v_heads;
  a.k_dim = (int)k_dim; a.v_dim = (int)v_dim; a.v_pad = (int)value_width(v_dim);
  a.chunks = chunk_count(seq);
  a.scale = scale;
  return a;
}
template <typename T>
void place_space(delta::Args<T>& a, const Space& w, char* ws) {
  a.keys = (uint16_t*)(ws + w.keys);
  a.tri = (uint16_t*)(ws + w.tri);
  a.zeros = (uint16_t*)(ws + w.zeros);
  a.vec = (float*)(ws + w.vec);
}

}  // namespace

#define MQC_BY_DTYPE(F)                    \
  switch (dtype) {                         \
    case MQC_F32: return F(float);         \
    case MQC_BF16: return F(bf16_t);       \
    default: return F(f16_t);              \
  }

extern "C" int mqc_gated_delta_chunk(void) { return delta::kC; }
extern "C" int64_t mqc_gated_delta_key_width(int64_t k_dim) {
  return k_dim < 1 ? MQC_E_SHAPE : k_dim > delta::kMaxK ? MQC_E_LIMIT : key_width(k_dim);
}
extern "C" int64_t mqc_gated_delta_value_width(int64_t v_dim) {
  return v_dim < 1 ? MQC_E_SHAPE : value_width(v_dim);
}

extern "C" int64_t mqc_gated_delta_workspace_bytes(int64_t batch, int64_t seq_len, int64_t k_heads,
                                                   int64_t v_heads, int64_t k_dim, int64_t v_dim,
                                                   int dtype, int backward) {
  const int st = shape(batch, seq_len, k_heads, v_heads, k_dim, v_dim, dtype, MQC_F32, MQC_F32,
                       backward != 0);
  if (st != MQC_OK) return st;
  return space(batch, seq_len, k_heads, v_heads, k_dim, v_dim, dtype, backward != 0).bytes;
}

extern "C" int mqc_gated_delta_fwd(const void* q, const void* k, const void* v, const int64_t* strides,
                                   const void* log_decay, int decay_dtype, const void* beta,
                                   int beta_dtype, const void* reset, const float* h0, void* o,
                                   float* h_last, float* states, float* residuals, int64_t batch,
                                   int64_t seq_len, int64_t k_heads, int64_t v_heads, int64_t k_dim,
                                   int64_t v_dim, float scale, int dtype, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  const int st = shape(batch, seq_len, k_heads, v_heads, k_dim, v_dim, dtype, decay_dtype, beta_dtype,
                       states || residuals);
  if (st != MQC_OK) return st;
  if (batch == 0) return MQC_OK;
  if (seq_len > 0 && (!q || !k || !v || !strides || !log_decay || !beta || !o || !workspace))
    return MQC_E_NULL;
  if (seq_len == 0 && !h_last) return MQC_OK;
  const Space w = space(batch, seq_len, k_heads, v_heads, k_dim, v_dim, dtype, false);
  if (workspace_bytes < w.bytes) return MQC_E_SPACE;
  if (!aligned(workspace, 16) || !aligned(states, 16) || !aligned(residuals, 16)) return MQC_E_ALIGN;
  static const int64_t none[9] = {};
#define MQC_F(T)                                                                                  \
  [&] {                                                                                           \
    delta::Args<T> a = args<T>(q, k, v, strides ? strides : none, log_decay, decay_dtype, beta,   \
                               beta_dtype, batch, seq_len, k_heads, v_heads, k_dim, v_dim, scale); \
    a.reset = (const uint8_t*)reset; a.h0 = h0; a.o = (T*)o; a.h_last = h_last;                   \
    a.states = states; a.resid = residuals;                                                       \
    place_space(a, w, (char*)workspace);                                                          \
    return delta::launch_fwd<T>(a, (hipStream_t)stream);                                          \
  }()
  MQC_BY_DTYPE(MQC_F)
#undef MQC_F
}

extern "C" int mqc_gated_delta_bwd(const void* q, const void* k, const void* v, const int64_t* strides,
                                   const void* log_decay, int decay_dtype, const void* beta,
                                   int beta_dtype, const void* reset, const float* states,
                                   const float* residuals, const void* d_o, const float* dh_last,
                                   void* dq, void* dk, void* dv, void* dlog_decay, void* dbeta,
                                   float* dh0, int64_t batch, int64_t seq_len, int64_t k_heads,
                                   int64_t v_heads, int64_t k_dim, int64_t v_dim, float scale,
                                   int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int st = shape(batch, seq_len, k_heads, v_heads, k_dim, v_dim, dtype, decay_dtype, beta_dtype, true);
  if (st != MQC_OK) return st;
  if (batch < 1 || seq_len < 1) return MQC_E_SHAPE;
  if (!q || !k || !v || !strides || !log_decay || !beta || !states || !residuals || !d_o || !dq || !dk ||
      !dv || !dlog_decay || !dbeta || !workspace)
    return MQC_E_NULL;
  const Space w = space(batch, seq_len, k_heads, v_heads, k_dim, v_dim, dtype, true);
  if (workspace_bytes < w.bytes) return MQC_E_SPACE;
  if (!aligned(workspace, 16) || !aligned(states, 16) || !aligned(residuals, 16)) return MQC_E_ALIGN;
#define MQC_F(T)                                                                                   \
  [&] {                                                                                            \
    delta::Args<T> a = args<T>(q, k, v, strides, log_decay, decay_dtype, beta, beta_dtype, batch,  \
                               seq_len, k_heads, v_heads, k_dim, v_dim, scale);                    \
    char* ws = (char*)workspace;                                                                   \
    a.reset = (const uint8_t*)reset;                                                               \
    a.states = const_cast<float*>(states); a.resid = const_cast<float*>(residuals);                \
    a.d_o = (const T*)d_o; a.dh_last = dh_last; a.dh0 = dh0;                                       \
    a.dq = (T*)dq; a.dk = (T*)dk; a.dv = (T*)dv; a.dg = dlog_decay; a.dbeta = dbeta;               \
    place_space(a, w, ws);                                                                         \
    a.dstates = (float*)(ws + w.dstates); a.z = (float*)(ws + w.z);                                \
    a.dq_part = (float*)(ws + w.dq); a.dk_part = (float*)(ws + w.dk);                              \
    return delta::launch_bwd<T>(a, (hipStream_t)stream);                                           \
  }()
  MQC_BY_DTYPE(MQC_F)
#undef MQC_F
}

extern "C" int mqc_gated_delta_step(const void* q, const void* k, const void* v, const int64_t* strides,
                                    const void* log_decay, int decay_dtype, const void* beta,
                                    int beta_dtype, float* h, void* o, int64_t batch, int64_t k_heads,
                                    int64_t v_heads, int64_t k_dim, int64_t v_dim, float scale,
                                    int dtype, void* stream) {
  const int st = shape(batch, 1, k_heads, v_heads, k_dim, v_dim, dtype, decay_dtype, beta_dtype, false);
  if (st != MQC_OK) return st;
  if (batch == 0) return MQC_OK;
  if (!q || !k || !v || !strides || !log_decay || !beta || !h || !o) return MQC_E_NULL;
#define MQC_F(T)                                                                                  \
  [&] {                                                                                           \
    delta::Args<T> a = args<T>(q, k, v, strides, log_decay, decay_dtype, beta, beta_dtype, batch, 1, \
                               k_heads, v_heads, k_dim, v_dim, scale);                            \
    a.o = (T*)o;                                                                                  \
    return delta::launch_step<T>(a, h, (hipStream_t)stream);                                      \
  }()
  MQC_BY_DTYPE(MQC_F)
#undef MQC_F
}
