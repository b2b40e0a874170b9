#pragma once
// The gated delta rule, a linear recurrence whose state is a matrix S [k_dim, v_dim] for each head:
//   p_t = a_t S_{t-1},  r_t = v_t - p_t^T k_t,  S_t = p_t + beta_t k_t r_t^T,  o_t = scale S_t^T q_t
// with a_t = exp(g_t), and a_t = 0 at the first token of a packed document.
//
// Tokens go in chunks of 64. With G the running sum of g in a chunk, D_ij = exp(G_i - G_j) for j <= i of
// one document (else 0) and e_i = exp(G_i) where nothing cut i off from the chunk's start (else 0):
//   R = V - e (K S),  r = T R with T = (I + A)^-1, A_ij = D_ij (k_i . k_j) beta_j for j < i,  u = beta r
//   O = scale (e (Q S) + P u),  P_ij = D_ij (q_i . k_j),   S' = e_63 S + K^T (D_63 u)
// Backward, from dO and dS' (T~ = (I + A~)^-1, A~_ij = beta_i D_ij (k_i . k_j)):
//   du = scale P^T dO + D_63 (K dS'),  z = T~^T du,  dv = beta z,  dbeta = z . r
//   dS = e_63 dS' + Q^T (scale e dO) - K^T (e beta z)
//   dQ = scale e (S dO^T)^T + (D dP) K with dP = scale dO u^T,  M = -beta_i D (z u^T) below the diagonal,
//   dK = [M K - e beta (S z^T)^T] + [(D dP)^T Q + M^T K + D_63 (dS' u^T)^T]
//   dg_t = sum over j < t <= i of W_ij, with W_ij = (D dP)_ij (q_i . k_j) + M_ij (k_i . k_j),
//     + sum over i >= t of e_i (scale q_i . (S dO_i) - beta_i k_i . (S z_i))
//     + sum over j < t of D_63,j k_j . (dS' u_j) + e_63 <dS', S>
// Every term of dg_t has the factor exp(g_t). (As sums from t on of q_i . dQ_i + k_i . dK_i, signs by bracket,
// which are the same, terms without it cancel: below g_t = -13 or so nothing but their rounding was left.)
//
// Three kinds of kernels. One over all chunks side by side forms the products within them (gram
// matrices, the triangular inverse) and lays every operand out as the matrix instructions read it. One
// walks the chunks of a head: columns of S do not depend on one another, so a workgroup has 16 or 32 of
// them, in registers from the first chunk to the last. What a product leaves (a column a lane, four rows
// each) is what the next one takes as its right operand if the left one's columns are in the order that
// place() gives. The backward's gradients of q, k, g and beta need
// sums over v_dim: again over all chunks side by side.
//
// Products are of bf16 matrix instructions on operands cut into pieces of 8 bits: three hold an fp32
// value whole, and two an fp16 one; of products of pieces those of 2^-24 and less are left out. What
// a 16-bit input enters as is exact; all else is held in 32 bits.
#include "common.hpp"

namespace mqc {
namespace delta {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kC = 64;          // tokens of a chunk
constexpr int kTri = 6;         // fragments of a triangular 64 x 64 matrix (rows of 16, columns of 32)
constexpr int kPieces = 3;      // of an fp32 value
constexpr int kMaxK = 128;      // k_dim

template <typename T>
constexpr int kIn = std::is_same<T, bf16_t>::value ? 1 : std::is_same<T, f16_t>::value ? 2 : 3;

// A fragment is 64 lanes x 16 bytes: what one matrix instruction takes of 16 rows (or columns) by 32.
// Lane 16 g + m holds row m; its eight columns are, of the 32, those that place(g, 0..7) names.
constexpr int kFrag = 512;  // 16-bit elements of a fragment
__device__ __host__ inline constexpr int place(int g, int j) { return (j >> 2) * 16 + 4 * g + (j & 3); }
// The inverse: the lane's g and the element j of column c of 32.
__device__ inline int place_g(int c) { return (c & 15) >> 2; }
__device__ inline int place_j(int c) { return (c >> 4) * 4 + (c & 3); }

// Eight values as N pieces: the leading ones cut off (a value less its cut part is exact), the last one
// rounded.
__device__ inline uint32_t cut2(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ inline float rest(float v) { return v - __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
template <int N>
__device__ inline void split(float (&x)[8], bf16x8 (&out)[N]) {
#pragma unroll
  for (int p = 0; p < N; ++p) {
    u32x4 w;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      w[c] = p + 1 < N ? cut2(x[2 * c], x[2 * c + 1]) : pack2<bf16_t>(x[2 * c], x[2 * c + 1]);
    out[p] = __builtin_bit_cast(bf16x8, w);
    if (p + 1 < N) {
#pragma unroll
      for (int c = 0; c < 8; ++c) x[c] = rest(x[c]);
    }
  }
}
template <int N>
__device__ inline void split(const floatx4& a, const floatx4& b, bf16x8 (&out)[N]) {
  float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  split<N>(x, out);
}

// acc += a b, the smallest products first.
template <int NA, int NB>
__device__ inline floatx4 mma(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], floatx4 acc) {
#pragma unroll
  for (int order = kPieces - 1; order >= 0; --order)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (order - i >= 0 && order - i < NB)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[order - i], acc, 0, 0, 0);
  return acc;
}

// After the last product into v and before v is used: eight wait states in the same basic block. (The
// compiler keeps results of matrix instructions from being read too early, but not in every case where a
// branch lies between the two: it read the last of four values before its sum was there.)
__device__ inline floatx4 settled(floatx4 v) {
  asm volatile("s_nop 7" : "+v"(v));
  return v;
}

// The same for the fp32 instruction, whose result takes 32 cycles.
__device__ inline floatx4 settled32(floatx4 v) {
  asm volatile("s_nop 15" : "+v"(v));
  return v;
}

template <int N>
__device__ inline void load_frag(const uint16_t* at, int lane, bf16x8 (&f)[N]) {
#pragma unroll
  for (int p = 0; p < N; ++p)
    f[p] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(at + p * kFrag + lane * 8));
}
template <int N>
__device__ inline void store_frag(uint16_t* at, int lane, const bf16x8 (&f)[N]) {
#pragma unroll
  for (int p = 0; p < N; ++p)
    *reinterpret_cast<u32x4*>(at + p * kFrag + lane * 8) = __builtin_bit_cast(u32x4, f[p]);
}

// The fragment of rows 16 mt and columns 32 s of a lower (upper) triangular matrix, -1 where it is zero.
__device__ __host__ inline constexpr int lower_frag(int mt, int s) {
  return mt < 2 ? (s ? -1 : mt) : 2 * mt - 2 + s;
}
__device__ __host__ inline constexpr int upper_frag(int mt, int s) {
  return mt < 2 ? 2 * mt + s : (s ? mt + 2 : -1);
}

template <typename T>
struct Args {
  const T *q, *k, *v;
  int64_t q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h;  // elements between batch rows, tokens, heads
  const void *g, *beta;                                 // [batch, seq, v_heads], of these types
  int g_type, beta_type;
  const uint8_t* reset;  // [batch, seq], or NULL
  const float* h0;       // [batch, v_heads, k_dim, v_dim], or NULL
  int64_t batch, seq, k_heads, v_heads;
  int k_dim, v_dim, v_pad;
  int64_t chunks;
  float scale;
  // The operands as fragments: of each key head and chunk K, K^T and Q (or, for the backward, Q^T), of
  // each value head and chunk T and P (or T~^T and P^T), and four vectors: e, D_63, beta, and the number
  // of documents begun since the chunk's start.
  uint16_t *keys, *tri, *zeros;  // (zeros: one fragment's pieces)
  float* vec;  // [batch, v_heads, chunks, 4, 64]
  // forward
  T* o;
  float *h_last, *states, *resid;  // states [.., chunks, KD, v_pad] and r [.., chunks, 64, v_pad], or NULL
  // backward
  const T* d_o;
  const float* dh_last;
  float *dstates, *z, *dh0;  // dstates as states, z as r
  T *dq, *dk, *dv;
  float *dq_part, *dk_part;  // [batch, seq, v_heads, k_dim] where value heads share a key head
  void *dg, *dbeta;
};

__device__ inline float load_any(const void* p, int64_t i, int type) {
  if (type == MQC_F32) return static_cast<const float*>(p)[i];
  return type == MQC_BF16 ? load_scalar(static_cast<const bf16_t*>(p) + i)
                          : load_scalar(static_cast<const f16_t*>(p) + i);
}
__device__ inline void store_any(void* p, int64_t i, int type, float v) {
  if (type == MQC_F32) static_cast<float*>(p)[i] = v;
  else if (type == MQC_BF16) store_scalar(static_cast<bf16_t*>(p) + i, v);
  else store_scalar(static_cast<f16_t*>(p) + i, v);
}

// Eight elements of a row as place(g, ..) of columns 32 s names them, zero past `dim`.
template <typename T>
__device__ inline void load_row8(const T* row, int s, int g, int dim, float (&x)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int at = 32 * s + 16 * half + 4 * g;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (at < dim) load_part(row, at, dim - at, v);
#pragma unroll
    for (int c = 0; c < 4; ++c) x[4 * half + c] = v[c];
  }
}

__device__ inline int64_t xcd_order(int64_t lin, int64_t n) {
  return n % kXCDs ? lin : (lin % kXCDs) * (n / kXCDs) + lin / kXCDs;
}

// The gates of a chunk, lane t of a wave its token t: beta, the documents begun since the chunk's start,
// and G in 64 bits (differences of long sums). Tokens past the end neither decay nor write.
struct Gates {
  float beta;
  int doc;
  double G;
};
template <typename T>
__device__ inline Gates chunk_gates(const Args<T>& a, int64_t b, int64_t hv, int64_t t0) {
  const int lane = threadIdx.x & 63;
  const int64_t t = t0 + lane, at = (b * a.seq + t) * a.v_heads + hv;
  const bool in = t < a.seq;
  float g = in ? load_any(a.g, at, a.g_type) : 0.f;
  if (g < -1e4f) g = -1e4f;  // exp is 0 from -104 on, and -inf has differences that are NaN
  Gates r;
  r.beta = in ? load_any(a.beta, at, a.beta_type) : 0.f;
  const bool first = in && a.reset && a.reset[b * a.seq + t] != 0;
  const uint64_t cuts = __ballot(first);
  r.doc = __popcll(cuts & (~0ull >> (63 - lane)));
  r.G = first ? 0.f : g;  // sums are a document's own, and nothing decays into its first token
#pragma unroll
  for (int n = 1; n < 64; n *= 2) {
    const double before = __shfl_up(r.G, n);
    const int other = __shfl_up(r.doc, n);
    if (lane >= n && other == r.doc) r.G += before;
  }
  return r;
}

// ---------------------------------------------------------------------------
// The products within chunks. A workgroup of four waves takes a chunk of a key head and of the value heads
// that share it; wave w rows 16 w.., whose gram products stay in its registers. Of 1536 chunks of 128 keys
// in bf16 49 us (the backward's operands 53): 32 KB read and 84 written of each, 3.6 TB/s.
// ---------------------------------------------------------------------------
template <typename T, int KD>
struct PrepShared {
  uint16_t frags[KD / 8 * kIn<T> * kFrag];  // K by rows; then Q, to be turned
  float m[kC][kC + 4], inv[kC][kC + 4];     // (rows at multiples of 16 bytes)
  double G[kC];
  float beta[kC];
  int doc[kC];
};

// 16 x 16 x 4 in fp32: lane 16 g + m holds a's row m, b's column m and of both the columns (rows) that it
// takes as number g.
__device__ inline floatx4 mma32(float a, float b, floatx4 acc) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, acc, 0, 0, 0);
}

// X = (I + m)^-1 for a strictly lower triangular m: its diagonal blocks of 16 by substitution, a column to a
// lane (products of powers of m would lose digits where keys repeat), then block diagonal by block diagonal,
// X_ij = -X_ii Y with Y = sum over j <= l < i of m_il X_lj, wave i. A sum over the 16 of a block takes them in
// the order 4 g + r, r = 0..3, in which Y leaves its product. Everything in fp32.
template <typename S>
__device__ inline void invert(S& s) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, o = 16 * w, g = lane >> 4, c = lane & 15;
  {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == c ? 1.f : 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (4 * q >= i) continue;
        const floatx4 row = *reinterpret_cast<const floatx4*>(&s.m[o + i][o + 4 * q]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (4 * q + j < i) v = fmaf(-row[j], x[4 * q + j], v);
      }
      x[i] = i < c ? 0.f : v;  // (a NaN of rows in between is none above the diagonal)
    }
    if (g == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s.inv[o + i][o + c] = x[i];
    }
  }
  __syncthreads();
  const floatx4 own = *reinterpret_cast<const floatx4*>(&s.inv[o + c][o + 4 * g]);  // X_ii
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    if (w >= d) {
      const int j = 16 * (w - d);
      floatx4 y = {};
#pragma unroll
      for (int n = 0; n < d; ++n) {
        const int l = j + 16 * n;
        const floatx4 left = *reinterpret_cast<const floatx4*>(&s.m[o + c][l + 4 * g]);
#pragma unroll
        for (int r = 0; r < 4; ++r) y = mma32(left[r], s.inv[l + 4 * g + r][j + c], y);
      }
      y = settled32(y);
      floatx4 x = {};
#pragma unroll
      for (int r = 0; r < 4; ++r) x = mma32(-own[r], y[r], x);
      x = settled32(x);
#pragma unroll
      for (int r = 0; r < 4; ++r) s.inv[o + 4 * g + r][j + c] = x[r];
    }
    __syncthreads();
  }
}

// K or Q, by rows in `frags`, by columns into `to`.
template <typename T, int KD>
__device__ inline void write_turned(const uint16_t* frags, uint16_t* to) {
  constexpr int NP = kIn<T>;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4;
  for (int f = w; f < KD / 8; f += 4) {
    const int d = f / 2 * 16 + (lane & 15), s = f & 1;
    const int c = d & 31, mine = place_g(c) * 16 * 8 + place_j(c);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = 32 * s + place(g, j);
        const uint32_t e = frags[((d / 32 * 4 + t / 16) * NP + p) * kFrag + (t & 15) * 8 + mine];
        v[j / 2] = j % 2 ? v[j / 2] | e << 16 : e;
      }
      *reinterpret_cast<u32x4*>(to + (f * NP + p) * kFrag + lane * 8) = v;
    }
  }
}

template <typename T, int KD, bool BWD>
__global__ __launch_bounds__(256) void delta_prep_kernel(Args<T> a) {
  constexpr int NP = kIn<T>, KS = KD / 32;
  __shared__ __attribute__((aligned(16))) PrepShared<T, KD> s;
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = blockIdx.x, chunk = unit % a.chunks, bh = unit / a.chunks;
  const int64_t b = bh / a.k_heads, hk = bh % a.k_heads, t0 = chunk * kC, t = t0 + 16 * w + m;
  const int group = (int)(a.v_heads / a.k_heads);
  uint16_t* keys = a.keys + unit * (3 * KD / 8 * NP * kFrag);
  constexpr int kPart = KD / 8 * NP * kFrag;
  if (unit == 0 && w < kPieces) *reinterpret_cast<u32x4*>(a.zeros + w * kFrag + lane * 8) = (u32x4){};
  // The gates of a value head, by one wave.
  const auto gates = [&](int64_t hv) {
    const Gates x = chunk_gates(a, b, hv, t0);
    s.G[lane] = x.G;
    s.beta[lane] = x.beta;
    s.doc[lane] = x.doc;
    const double end = __shfl(x.G, 63);
    float* vec = a.vec + ((b * a.v_heads + hv) * a.chunks + chunk) * 4 * kC;
    vec[lane] = x.doc == 0 ? expf((float)x.G) : 0.f;
    vec[kC + lane] = x.doc == __shfl(x.doc, 63) ? expf((float)(end - x.G)) : 0.f;
    vec[2 * kC + lane] = x.beta;
    vec[3 * kC + lane] = (float)x.doc;
  };

  // Rows of K and Q as fragments.
  bf16x8 kf[KS][NP], qf[KS][NP];
  {
    const T* krow = a.k + b * a.k_b + t * a.k_t + hk * a.k_h;
    const T* qrow = a.q + b * a.q_b + t * a.q_t + hk * a.q_h;
    const int dim = t < a.seq ? a.k_dim : 0;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      float x[8], y[8];
      load_row8(krow, i, g, dim, x);
      load_row8(qrow, i, g, dim, y);
      split<NP>(x, kf[i]);
      split<NP>(y, qf[i]);
    }
  }
  if (w == 3) gates(hk * group);
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    const int at = (i * 4 + w) * NP * kFrag;
    store_frag(s.frags + at, lane, kf[i]);
    const int to = (w * KS + i) * NP * kFrag;  // a wave of the walk reads its own together
    store_frag(keys + to, lane, kf[i]);
    if constexpr (!BWD) store_frag(keys + 2 * kPart + to, lane, qf[i]);
  }
  __syncthreads();
  floatx4 kk[4] = {}, qk[4] = {};
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    if (n > w) continue;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      bf16x8 kn[NP];
      load_frag(s.frags + (i * 4 + n) * NP * kFrag, lane, kn);
      kk[n] = mma(kf[i], kn, kk[n]);
      qk[n] = mma(qf[i], kn, qk[n]);
    }
    kk[n] = settled(kk[n]), qk[n] = settled(qk[n]);
  }
  write_turned<T, KD>(s.frags, keys + kPart);
  if constexpr (BWD) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KS; ++i) store_frag(s.frags + (i * 4 + w) * NP * kFrag, lane, qf[i]);
    __syncthreads();
    write_turned<T, KD>(s.frags, keys + 2 * kPart);
  }

  for (int j = 0; j < group; ++j) {
    const int64_t hv = hk * group + j, at = (b * a.v_heads + hv) * a.chunks + chunk;
    if (j > 0) {
      __syncthreads();  // the head before is done with what follows
      if (w == 3) gates(hv);
      __syncthreads();
    }
    // m, and P in registers (above the diagonal nothing is read).
    floatx4 P[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      P[n] = (floatx4){};
      if (n > w) continue;
      const int col = 16 * n + m;
      const double Gc = s.G[col];
      const int dc = s.doc[col];
      const float bc = s.beta[col];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * w + 4 * g + r;
        const bool seen = (col <= row) & (s.doc[row] == dc);
        const float gap = (float)(s.G[row] - Gc);
        const float D = expf(seen ? gap : -1e4f);  // else 0
        const float by = D * (BWD ? s.beta[row] : bc);
        s.m[row][col] = (seen & (col < row)) ? by * kk[n][r] : 0.f;
        P[n][r] = seen ? D * qk[n][r] : 0.f;
      }
    }
    __syncthreads();
    invert(s);
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (n <= w) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s.m[16 * w + 4 * g + r][16 * n + m] = P[n][r];
      }
    __syncthreads();
    uint16_t* tri = a.tri + at * (2 * kTri * kPieces * kFrag);
    for (int f = w; f < 2 * kTri; f += 4) {
      const int n = f % kTri;  // which rows of 16 and columns of 32
      const int mt = BWD ? (n < 4 ? n / 2 : n - 2) : (n < 2 ? n : n / 2 + 1);
      const int ks = BWD ? (n < 4 ? n % 2 : 1) : (n < 2 ? 0 : n % 2);
      const float(*from)[kC + 4] = f < kTri ? s.inv : s.m;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = 16 * mt + m, col = 32 * ks + place(g, e);
        const int i = BWD ? col : row, l = BWD ? row : col;
        // Not of another document (whose NaN may have come here) and not above the diagonal.
        x[e] = l > i || s.doc[i] != s.doc[l] ? 0.f : from[i][l];
      }
      bf16x8 p[kPieces];
      split<kPieces>(x, p);
      store_frag(tri + f * kPieces * kFrag, lane, p);
    }
  }
}

// ---------------------------------------------------------------------------
// The walks. A workgroup has CT times 16 columns of a head's state, its wave w the tokens 16 w.. of each
// chunk and the state's rows 16 w.. and 16 (w + 4)... A product's left operand is the wave's own rows, from
// memory to registers a chunk ahead; its right one (the state, then what the tokens leave) is all waves',
// and goes through LDS as pieces. A chunk waits for the one before, three barriers each: with a workgroup to
// a CU for 2.3 us (128 keys, bf16), of which matrix instructions take 0.4 and vector instructions 0.75. With
// operands brought to LDS by a workgroup of one wave each it was 12.
// ---------------------------------------------------------------------------
template <int KD, int CT>
struct WalkShared {
  static constexpr int KS = KD / 32;
  uint16_t state[2][CT][KS * kPieces * kFrag];  // of this chunk and of the next
  uint16_t x[CT][2 * kPieces * kFrag], u[CT][2 * kPieces * kFrag], y[CT][2 * kPieces * kFrag];
  uint16_t d_o[2][CT][2 * kPieces * kFrag];     // (backward)
  float xs[2][CT][kC][16];                      // x and u in fp32 where documents meet
  int bad[2][CT][4];                            // whether a wave has some that are not finite
};

// A barrier for what is in LDS; accesses to memory stay under way.
__device__ inline void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Rows 16 tile.. of a right operand [.., 16], as pieces of its fragments.
template <int N>
__device__ inline void put_tile(uint16_t* frags, int tile, const floatx4& v) {
  const int lane = threadIdx.x & 63;
  float x[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int p = 0; p < N; ++p) {
    uint2 w;
    w.x = p + 1 < N ? cut2(x[0], x[1]) : pack2<bf16_t>(x[0], x[1]);
    w.y = p + 1 < N ? cut2(x[2], x[3]) : pack2<bf16_t>(x[2], x[3]);
    *reinterpret_cast<uint2*>(frags + (tile / 2 * N + p) * kFrag + lane * 8 + tile % 2 * 4) = w;
    if (p + 1 < N) {
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = rest(x[c]);
    }
  }
}

// Element (row, col) of a triangular matrix that is there as fragments.
template <bool UPPER>
__device__ inline float tri_at(const uint16_t* tri, int row, int col) {
  const int f = UPPER ? upper_frag(row / 16, col / 32) : lower_frag(row / 16, col / 32);
  const uint16_t* at = tri + f * kPieces * kFrag + (place_g(col & 31) * 16 + (row & 15)) * 8 +
                       place_j(col & 31);
  float v = 0.f;
#pragma unroll
  for (int p = kPieces - 1; p >= 0; --p) v += io<bf16_t>::bits_to_f32(at[p * kFrag]);
  return v;
}

__device__ inline bool finite(float v) { return fabsf(v) < __builtin_huge_valf(); }

// The wave's rows of a triangular matrix: fragments of its two columns of 32, one of which may be zero.
// (The zeros come from memory too: what is there already would be waited for.)
template <bool UPPER>
__device__ inline void load_tri(const uint16_t* tri, const uint16_t* zeros, int w,
                                bf16x8 (&f)[2][kPieces]) {
  const int lane = threadIdx.x & 63;
  const int first = UPPER ? (w < 2 ? 2 * w : w + 1) : (w < 2 ? w : 2 * w - 2);
  const uint16_t* at = tri + first * kPieces * kFrag;
  load_frag(UPPER && w >= 2 ? zeros : at, lane, f[0]);
  load_frag(!UPPER && w < 2 ? zeros : at + kPieces * kFrag, lane, f[1]);
}
// Their product with x.
template <int NX>
__device__ inline floatx4 tri_product(const bf16x8 (&f)[2][kPieces], const uint16_t* x) {
  const int lane = threadIdx.x & 63;
  floatx4 v[2] = {};
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    bf16x8 b[NX];
    load_frag(x + s * NX * kFrag, lane, b);
    v[s] = mma(f[s], b, v[s]);
  }
  return settled(v[0]) + settled(v[1]);
}
// The same where documents meet in the chunk and x is not finite somewhere (`bad`, of each wave): term by
// term, since zero times NaN is not zero.
template <bool UPPER>
__device__ inline bool tri_apart(const int* bad, const float (*xs)[16], const uint16_t* tri, const float* doc,
                                 int w, floatx4& out) {
  if (!(bad[0] | bad[1] | bad[2] | bad[3])) return false;
  const int lane = threadIdx.x & 63;
  for (int r = 0; r < 4; ++r) {
    const int row = 16 * w + 4 * (lane >> 4) + r;
    float s = 0.f;
#pragma unroll 1
    for (int j = UPPER ? row : 0; UPPER ? j < kC : j <= row; ++j)
      if (doc[j] == doc[row]) s = fmaf(tri_at<UPPER>(tri, row, j), xs[j][lane & 15], s);
    out[r] = s;
  }
  return true;
}

// What the two walks share: where a workgroup is, and its operands.
template <typename T, int KD, bool BWD, int CT>
struct Walker {
  static constexpr int NP = kIn<T>, KS = KD / 32, MT = KD / 16 > 4 ? 2 : 1;
  static constexpr int kPart = KD / 8 * NP * kFrag, kTriPart = kTri * kPieces * kFrag;
  const Args<T>& a;
  int lane, w, g, m;
  int64_t b, hv, hk, bh;
  int col0;
  bool holds;  // whether the wave has rows of the state (of 32 only two do)
  const uint16_t *keys, *tri;
  const float* vec;

  __device__ explicit Walker(const Args<T>& a_) : a(a_) {
    lane = threadIdx.x & 63;
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    g = lane >> 4, m = lane & 15;
    const int groups = (a.v_pad / 16 + CT - 1) / CT;
    const int64_t unit = xcd_order(blockIdx.x, gridDim.x);
    bh = unit / groups;
    b = bh / a.v_heads, hv = bh % a.v_heads, hk = hv / (a.v_heads / a.k_heads);
    col0 = (int)(unit % groups) * CT * 16;
    holds = w < KD / 16;
    keys = a.keys + (b * a.k_heads + hk) * a.chunks * (3 * kPart);
    tri = a.tri + bh * a.chunks * (2 * kTriPart);
    vec = a.vec + bh * a.chunks * (4 * kC);
  }
  __device__ int col(int ct) const { return col0 + 16 * ct + m; }
  // Fragments of the wave's tokens of K or Q, and of its rows of K^T or Q^T, of a chunk.
  __device__ const uint16_t* part(int64_t c, int i) const { return keys + c * (3 * kPart) + i * kPart; }
  __device__ void load_rows(int64_t c, int i, bf16x8 (&f)[KS][NP]) const {
#pragma unroll
    for (int s = 0; s < KS; ++s) load_frag(part(c, i) + (w * KS + s) * NP * kFrag, lane, f[s]);
  }
  __device__ void load_cols(int64_t c, int i, bf16x8 (&f)[MT][2][NP]) const {
    const int tile = holds ? w : 0;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        load_frag(part(c, i) + ((tile + 4 * t) * 2 + s) * NP * kFrag, lane, f[t][s]);
  }
  // rows x state (K's, and in the forward Q's too: each piece of the state is read once).
  __device__ floatx4 row_product(const bf16x8 (&f)[KS][NP], const uint16_t* state) const {
    floatx4 v[2] = {};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      bf16x8 b[kPieces];
      load_frag(state + s * kPieces * kFrag, lane, b);
      v[s % 2] = mma(f[s], b, v[s % 2]);
    }
    return KS > 1 ? settled(v[0]) + settled(v[1]) : settled(v[0]);
  }
  __device__ void row_products(const bf16x8 (&f)[KS][NP], const bf16x8 (&h)[KS][NP], const uint16_t* state,
                               floatx4& x, floatx4& y) const {
    x = (floatx4){}, y = (floatx4){};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      bf16x8 b[kPieces];
      load_frag(state + s * kPieces * kFrag, lane, b);
      x = mma(f[s], b, x);
      y = mma(h[s], b, y);
    }
    x = settled(x), y = settled(y);
  }
  // S += cols x.
  __device__ void col_product(const bf16x8 (&f)[MT][2][NP], const uint16_t* x, floatx4 (&S)[MT]) const {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 xf[kPieces];
      load_frag(x + s * kPieces * kFrag, lane, xf);
#pragma unroll
      for (int t = 0; t < MT; ++t) S[t] = mma(f[t][s], xf, S[t]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) S[t] = settled(S[t]);
  }
  // The columns of tokens of other documents than `keep` as zero.
  __device__ void cut_cols(bf16x8 (&f)[MT][2][NP], const float* doc, float keep) const {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 mask = {};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (doc[32 * s + place(g, j)] == keep) mask[j / 2] |= j % 2 ? 0xffff0000u : 0xffffu;
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int p = 0; p < NP; ++p)
          f[t][s][p] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, f[t][s][p]) & mask);
    }
  }
  __device__ void put_state(uint16_t* frags, const floatx4 (&S)[MT]) const {
    if (!holds) return;
#pragma unroll
    for (int t = 0; t < MT; ++t) put_tile<kPieces>(frags, w + 4 * t, S[t]);
  }
  // The wave's rows of a state [k_dim, v_dim] in memory.
  __device__ void load_state(const float* from, int ct, floatx4 (&S)[MT]) const {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * (w + 4 * t) + 4 * g + r;
        S[t][r] = from && d < a.k_dim && col(ct) < a.v_dim
                      ? from[(bh * a.k_dim + d) * a.v_dim + col(ct)] : 0.f;
      }
  }
  __device__ void store_state(float* to, int ct, const floatx4 (&S)[MT]) const {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * (w + 4 * t) + 4 * g + r;
        if (d < a.k_dim && col(ct) < a.v_dim) to[(bh * a.k_dim + d) * a.v_dim + col(ct)] = S[t][r];
      }
  }
  // The same between chunks, padded.
  __device__ void store_padded(float* to, int64_t c, int ct, const floatx4 (&S)[MT]) const {
    if (!holds || col(ct) >= a.v_pad) return;
    float* base = to + (bh * a.chunks + c) * KD * a.v_pad;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        base[(uint32_t)((16 * (w + 4 * t) + 4 * g + r) * a.v_pad + col(ct))] = S[t][r];
  }
  __device__ void store_rows(float* to, int64_t c, int ct, const floatx4& v) const {
    if (col(ct) >= a.v_pad) return;
    float* base = to + (bh * a.chunks + c) * kC * a.v_pad;
#pragma unroll
    for (int r = 0; r < 4; ++r) base[(uint32_t)((16 * w + 4 * g + r) * a.v_pad + col(ct))] = v[r];
  }
  __device__ bool here(int64_t c, int r) const { return c * kC + 16 * w + 4 * g + r < a.seq; }
  __device__ bool whole(int64_t c) const { return (c + 1) * kC <= a.seq && col0 + 16 * CT <= a.v_dim; }
  __device__ float tile_value(const T (&v)[4], int64_t c, int ct, int r) const {
    return here(c, r) && col(ct) < a.v_dim ? load_scalar(&v[r]) : 0.f;
  }
  // Rows that are not finite, for tri_product.
  __device__ void mark(float (*xs)[16], int* bad, const floatx4& v) const {
    bool ok = true;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      xs[16 * w + 4 * g + r][m] = v[r];
      ok = ok && finite(v[r]);
    }
    const bool some = __ballot(!ok) != 0;
    if (lane == 0) bad[w] = some;
  }
};

// The wave's tokens of v (or dO), and of o (or dv): elements of a chunk from its first token, 16 columns.
template <typename T>
struct TileRows {
  T* first;       // of the head
  int64_t token;  // elements between tokens
  int64_t at[4];  // of the lane's four in a chunk, at its column
  __device__ TileRows(T* x, int64_t token_, int w, int g, int col) : first(x), token(token_) {
#pragma unroll
    for (int r = 0; r < 4; ++r) at[r] = (16 * w + 4 * g + r) * token_ + col;
  }
  // (of `whole` chunks; else past the ends the last token's and the last column)
  template <typename V, typename K>
  __device__ void load(const K& k, int64_t c, int ct, V (&v)[4]) const {
    if (k.whole(c)) {
      const T* base = first + c * kC * token + 16 * ct;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = base[at[r]];
    } else {
      const int col = k.col(ct) < k.a.v_dim ? k.col(ct) : k.a.v_dim - 1;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t t = c * kC + 16 * k.w + 4 * k.g + r;
        v[r] = first[(t < k.a.seq ? t : k.a.seq - 1) * token + col];
      }
    }
  }
  template <typename K>
  __device__ void store(const K& k, int64_t c, int ct, const floatx4& v) const {
    T* base = first + c * kC * token + 16 * ct;
    if (k.whole(c)) {
#pragma unroll
      for (int r = 0; r < 4; ++r) store_scalar(base + at[r], v[r]);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (k.here(c, r) && k.col(ct) < k.a.v_dim) store_scalar(base + at[r], v[r]);
    }
  }
};

// A chunk's gates, for the wave's tokens.
struct RowGates {
  floatx4 e, end, beta, doc;
  float all, first, last;
  __device__ void load(const float* vec, int w, int g) {
    const int at = 16 * w + 4 * g;
    e = *reinterpret_cast<const floatx4*>(vec + at);
    end = *reinterpret_cast<const floatx4*>(vec + kC + at);
    beta = *reinterpret_cast<const floatx4*>(vec + 2 * kC + at);
    doc = *reinterpret_cast<const floatx4*>(vec + 3 * kC + at);
    all = vec[kC - 1], first = vec[3 * kC], last = vec[4 * kC - 1];
  }
};

// Waves to a SIMD where their operands leave registers for that (two hide one another's waits: 384 workgroups
// of 32 chunks walk forward in 159 us and back in 171).
template <typename T, int KD, int CT, bool BWD>
constexpr int kWalkWaves = CT == 1 && (BWD ? (kIn<T> == 1 && KD == 128) || (kIn<T> == 2 && KD < 128)
                                           : kIn<T> == 1 || (kIn<T> == 2 && KD < 128)) ? 2 : 1;

template <typename T, int KD, int CT>
__global__ __launch_bounds__(256, (kWalkWaves<T, KD, CT, false>)) void delta_fwd_kernel(Args<T> a) {
  __shared__ __attribute__((aligned(16))) WalkShared<KD, CT> s;
  using K = Walker<T, KD, false, CT>;
  const K k(a);
  constexpr int NP = K::NP, KS = K::KS, MT = K::MT;
  floatx4 S[CT][MT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    k.load_state(a.h0, ct, S[ct]);
    k.put_state(s.state[0][ct], S[ct]);
  }
  bf16x8 kf[KS][NP], qf[KS][NP], tf[2][kPieces], pf[2][kPieces], cf[MT][2][NP];
  T v[CT][4];
  const int64_t heads = a.v_heads * (int64_t)a.v_dim;
  const TileRows<const T> from(a.v + k.b * a.v_b + k.hv * a.v_h, a.v_t, k.w, k.g, k.col(0));
  const TileRows<T> to(a.o + k.b * a.seq * heads + k.hv * a.v_dim, heads, k.w, k.g, k.col(0));
  RowGates next;
  if (a.chunks > 0) {
    next.load(k.vec, k.w, k.g);
    k.load_rows(0, 0, kf);
    k.load_rows(0, 2, qf);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) from.load(k, 0, ct, v[ct]);
    load_tri<false>(k.tri, a.zeros, k.w, tf);
    k.load_cols(0, 1, cf);
    load_tri<false>(k.tri + K::kTriPart, a.zeros, k.w, pf);
  }
  for (int64_t c = 0; c < a.chunks; ++c) {
    // What comes next goes out as soon as its place is free (behind the last chunk, once more its own).
    const int64_t ahead = c + 1 < a.chunks ? c + 1 : c;
    const RowGates at = next;
    const float* doc = k.vec + c * 4 * kC + 3 * kC;
    const uint16_t *tri = k.tri + c * 2 * K::kTriPart, *tri_ahead = k.tri + ahead * 2 * K::kTriPart;
    const bool mixed = at.first != at.last, cut = at.last != 0.f;
    lds_barrier();
    next.load(k.vec + ahead * 4 * kC, k.w, k.g);
    floatx4 x[CT], qs[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) k.row_products(kf, qf, s.state[c & 1][ct], x[ct], qs[ct]);
    k.load_rows(ahead, 0, kf);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float vt = k.tile_value(v[ct], c, ct, r);
        x[ct][r] = at.doc[r] == 0.f && k.here(c, r) ? fmaf(-at.e[r], x[ct][r], vt) : vt;
      }
      put_tile<kPieces>(s.x[ct], k.w, x[ct]);
      if (mixed) k.mark(s.xs[0][ct], s.bad[0][ct], x[ct]);
    }
    lds_barrier();
    k.load_rows(ahead, 2, qf);
    floatx4 r[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      from.load(k, ahead, ct, v[ct]);
      if (!mixed || !tri_apart<false>(s.bad[0][ct], s.xs[0][ct], tri, doc, k.w, r[ct]))
        r[ct] = tri_product<kPieces>(tf, s.x[ct]);
      floatx4 u, y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[i] = r[ct][i] * at.beta[i];
        y[i] = at.doc[i] == at.last ? u[i] * at.end[i] : 0.f;
      }
      put_tile<kPieces>(s.u[ct], k.w, u);
      put_tile<kPieces>(s.y[ct], k.w, y);
      if (mixed) k.mark(s.xs[1][ct], s.bad[1][ct], u);
    }
    load_tri<false>(tri_ahead, a.zeros, k.w, tf);
    if (mixed) k.cut_cols(cf, doc, at.last);
    lds_barrier();
    if (a.states) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) k.store_padded(a.states, c, ct, S[ct]);
    }
    floatx4 o[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) S[ct][t][i] = cut ? 0.f : S[ct][t][i] * at.all;
      k.col_product(cf, s.y[ct], S[ct]);
      if (!mixed || !tri_apart<false>(s.bad[1][ct], s.xs[1][ct], tri + K::kTriPart, doc, k.w, o[ct]))
        o[ct] = tri_product<kPieces>(pf, s.u[ct]);
      k.put_state(s.state[(c + 1) & 1][ct], S[ct]);
    }
    k.load_cols(ahead, 1, cf);
    load_tri<false>(tri_ahead + K::kTriPart, a.zeros, k.w, pf);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[ct][i] = a.scale * (at.doc[i] == 0.f ? fmaf(at.e[i], qs[ct][i], o[ct][i]) : o[ct][i]);
      to.store(k, c, ct, o[ct]);
      if (a.resid) k.store_rows(a.resid, c, ct, r[ct]);
    }
  }
  if (a.h_last && k.holds) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) k.store_state(a.h_last, ct, S[ct]);
  }
}

// The same by eight waves, for workgroups that have a CU each: four take the state from chunk to chunk, and
// four make the outputs beside them, their products with the state while the tokens' x is made, those with
// what the tokens leave while the next state is. A chunk takes 1.95 us for 2.3 (96 workgroups, 128 keys,
// bf16); where two workgroups share a CU, four waves each are faster (384 of them: 162 us for 181).
template <typename T, int KD>
__global__ __launch_bounds__(512, 2) void delta_fwd_beside_kernel(Args<T> a) {
  __shared__ __attribute__((aligned(16))) WalkShared<KD, 1> s;
  using K = Walker<T, KD, false, 1>;
  const K k(a);
  constexpr int NP = K::NP, KS = K::KS, MT = K::MT;
  const auto ahead_of = [&](int64_t c) { return c + 1 < a.chunks ? c + 1 : c; };
  RowGates next;
  if (a.chunks > 0) next.load(k.vec, k.w, k.g);
  if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 8)) {
    bf16x8 qf[KS][NP], pf[2][kPieces];
    const int64_t heads = a.v_heads * (int64_t)a.v_dim;
    const TileRows<T> to(a.o + k.b * a.seq * heads + k.hv * a.v_dim, heads, k.w, k.g, k.col(0));
    if (a.chunks > 0) {
      k.load_rows(0, 2, qf);
      load_tri<false>(k.tri + K::kTriPart, a.zeros, k.w, pf);
    }
    for (int64_t c = 0; c < a.chunks; ++c) {
      const int64_t ahead = ahead_of(c);
      const RowGates at = next;
      const float* doc = k.vec + c * 4 * kC + 3 * kC;
      lds_barrier();
      next.load(k.vec + ahead * 4 * kC, k.w, k.g);
      const floatx4 qs = k.row_product(qf, s.state[c & 1][0]);
      k.load_rows(ahead, 2, qf);
      lds_barrier();
      lds_barrier();
      floatx4 o;
      if (at.first == at.last ||
          !tri_apart<false>(s.bad[1][0], s.xs[1][0], k.tri + (2 * c + 1) * K::kTriPart, doc, k.w, o))
        o = tri_product<kPieces>(pf, s.u[0]);
      load_tri<false>(k.tri + (2 * ahead + 1) * K::kTriPart, a.zeros, k.w, pf);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = a.scale * (at.doc[i] == 0.f ? fmaf(at.e[i], qs[i], o[i]) : o[i]);
      to.store(k, c, 0, o);
    }
    return;
  }
  floatx4 S[MT];
  k.load_state(a.h0, 0, S);
  k.put_state(s.state[0][0], S);
  bf16x8 kf[KS][NP], tf[2][kPieces], cf[MT][2][NP];
  T v[4];
  const TileRows<const T> from(a.v + k.b * a.v_b + k.hv * a.v_h, a.v_t, k.w, k.g, k.col(0));
  if (a.chunks > 0) {
    k.load_rows(0, 0, kf);
    from.load(k, 0, 0, v);
    load_tri<false>(k.tri, a.zeros, k.w, tf);
    k.load_cols(0, 1, cf);
  }
  for (int64_t c = 0; c < a.chunks; ++c) {
    const int64_t ahead = ahead_of(c);
    const RowGates at = next;
    const float* doc = k.vec + c * 4 * kC + 3 * kC;
    const bool mixed = at.first != at.last, cut = at.last != 0.f;
    lds_barrier();
    next.load(k.vec + ahead * 4 * kC, k.w, k.g);
    floatx4 x = k.row_product(kf, s.state[c & 1][0]);
    k.load_rows(ahead, 0, kf);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float vt = k.tile_value(v, c, 0, i);
      x[i] = at.doc[i] == 0.f && k.here(c, i) ? fmaf(-at.e[i], x[i], vt) : vt;
    }
    put_tile<kPieces>(s.x[0], k.w, x);
    if (mixed) k.mark(s.xs[0][0], s.bad[0][0], x);
    lds_barrier();
    from.load(k, ahead, 0, v);
    floatx4 r, u, y;
    if (!mixed || !tri_apart<false>(s.bad[0][0], s.xs[0][0], k.tri + 2 * c * K::kTriPart, doc, k.w, r))
      r = tri_product<kPieces>(tf, s.x[0]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = r[i] * at.beta[i];
      y[i] = at.doc[i] == at.last ? u[i] * at.end[i] : 0.f;
    }
    put_tile<kPieces>(s.u[0], k.w, u);
    put_tile<kPieces>(s.y[0], k.w, y);
    if (mixed) k.mark(s.xs[1][0], s.bad[1][0], u);
    load_tri<false>(k.tri + 2 * ahead * K::kTriPart, a.zeros, k.w, tf);
    if (mixed) k.cut_cols(cf, doc, at.last);
    lds_barrier();
    if (a.states) k.store_padded(a.states, c, 0, S);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[t][i] = cut ? 0.f : S[t][i] * at.all;
    k.col_product(cf, s.y[0], S);
    k.put_state(s.state[(c + 1) & 1][0], S);
    k.load_cols(ahead, 1, cf);
    if (a.resid) k.store_rows(a.resid, c, 0, r);
  }
  if (a.h_last && k.holds) k.store_state(a.h_last, 0, S);
}

template <typename T, int KD, int CT>
__global__ __launch_bounds__(256, (kWalkWaves<T, KD, CT, true>)) void delta_bwd_kernel(Args<T> a) {
  __shared__ __attribute__((aligned(16))) WalkShared<KD, CT> s;
  using K = Walker<T, KD, true, CT>;
  const K k(a);
  constexpr int NP = K::NP, KS = K::KS, MT = K::MT;
  const int64_t heads = a.v_heads * (int64_t)a.v_dim, end = a.chunks - 1;
  const int64_t first = k.b * a.seq * heads + k.hv * a.v_dim;
  const TileRows<const T> from(a.d_o + first, heads, k.w, k.g, k.col(0));
  const TileRows<T> to(a.dv + first, heads, k.w, k.g, k.col(0));
  const auto put_grad = [&](int64_t c, int ct, const T (&raw)[4], floatx4& v) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = k.tile_value(raw, c, ct, r);
    put_tile<NP>(s.d_o[c & 1][ct], k.w, v);
  };
  floatx4 S[CT][MT], v[CT];  // the gradient of the state after the chunk; the wave's tokens of dO
  T raw[CT][4];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    k.load_state(a.dh_last, ct, S[ct]);
    k.put_state(s.state[end & 1][ct], S[ct]);
    from.load(k, end, ct, raw[ct]);
    put_grad(end, ct, raw[ct], v[ct]);
  }
  bf16x8 kf[KS][NP], tf[2][kPieces], pf[2][kPieces], cf[MT][2][NP], qf[MT][2][NP];
  RowGates next;
  next.load(k.vec + end * 4 * kC, k.w, k.g);
  k.load_rows(end, 0, kf);
  load_tri<true>(k.tri + (2 * end + 1) * K::kTriPart, a.zeros, k.w, pf);
  load_tri<true>(k.tri + 2 * end * K::kTriPart, a.zeros, k.w, tf);
  k.load_cols(end, 2, qf);
  k.load_cols(end, 1, cf);
  for (int64_t c = end; c >= 0; --c) {
    const int64_t ahead = c > 0 ? c - 1 : 0;
    const RowGates at = next;
    const float* doc = k.vec + c * 4 * kC + 3 * kC;
    const uint16_t *tri = k.tri + c * 2 * K::kTriPart, *tri_ahead = k.tri + ahead * 2 * K::kTriPart;
    const bool mixed = at.first != at.last, cut = at.last != 0.f;
    if (mixed) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) k.mark(s.xs[1][ct], s.bad[1][ct], v[ct]);
    }
    if (cut) {
      k.cut_cols(qf, doc, 0.f);
      k.cut_cols(cf, doc, 0.f);
    }
    lds_barrier();
    next.load(k.vec + ahead * 4 * kC, k.w, k.g);
    floatx4 y[CT], z[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      from.load(k, ahead, ct, raw[ct]);
      y[ct] = k.row_product(kf, s.state[c & 1][ct]);
      if (!mixed || !tri_apart<true>(s.bad[1][ct], s.xs[1][ct], tri + K::kTriPart, doc, k.w, z[ct]))
        z[ct] = tri_product<NP>(pf, s.d_o[c & 1][ct]);
    }
    k.load_rows(ahead, 0, kf);
    load_tri<true>(tri_ahead + K::kTriPart, a.zeros, k.w, pf);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      floatx4 x;  // e dO, for the state
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        z[ct][r] *= a.scale;
        if (at.doc[r] == at.last) z[ct][r] = fmaf(at.end[r], y[ct][r], z[ct][r]);
        x[r] = at.doc[r] == 0.f ? v[ct][r] * (a.scale * at.e[r]) : 0.f;
      }
      put_tile<kPieces>(s.x[ct], k.w, z[ct]);
      put_tile<kPieces>(s.u[ct], k.w, x);
      if (mixed) k.mark(s.xs[0][ct], s.bad[0][ct], z[ct]);
    }
    lds_barrier();
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      k.store_padded(a.dstates, c, ct, S[ct]);
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[ct][t][r] = cut ? 0.f : S[ct][t][r] * at.all;
      if (!mixed || !tri_apart<true>(s.bad[0][ct], s.xs[0][ct], tri, doc, k.w, z[ct]))
        z[ct] = tri_product<kPieces>(tf, s.x[ct]);
      k.col_product(qf, s.u[ct], S[ct]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        y[ct][r] = at.beta[r] * z[ct][r];
        v[ct][r] = at.doc[r] == 0.f ? -y[ct][r] * at.e[r] : 0.f;
      }
      put_tile<kPieces>(s.y[ct], k.w, v[ct]);
    }
    load_tri<true>(tri_ahead, a.zeros, k.w, tf);
    k.load_cols(ahead, 2, qf);
    lds_barrier();
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      k.col_product(cf, s.y[ct], S[ct]);
      k.put_state(s.state[(c + 1) & 1][ct], S[ct]);
      put_grad(ahead, ct, raw[ct], v[ct]);
    }
    k.load_cols(ahead, 1, cf);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      k.store_rows(a.z, c, ct, z[ct]);
      to.store(k, c, ct, y[ct]);
    }
  }
  if (a.dh0 && k.holds) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) k.store_state(a.dh0, ct, S[ct]);
  }
}

// The same by eight waves (as forward): four take the state's gradient from chunk to chunk, and four bring them
// what does not depend on it, P^T dO of the next chunk and Q^T (e dO) of this one. In fp32 with 64 keys 105
// workgroups take 57 us for 84; 384 of them in bf16 183, with four waves 172.
template <int KD>
struct BesideShared {
  floatx4 z[4][64], s[KD / 16 > 4 ? 2 : 1][4][64];  // as the chain's waves hold z and the state
};
template <typename T, int KD>
__global__ __launch_bounds__(512, 2) void delta_bwd_beside_kernel(Args<T> a) {
  __shared__ __attribute__((aligned(16))) WalkShared<KD, 1> s;
  __shared__ BesideShared<KD> beside;
  using K = Walker<T, KD, true, 1>;
  const K k(a);
  constexpr int NP = K::NP, KS = K::KS, MT = K::MT;
  const int64_t heads = a.v_heads * (int64_t)a.v_dim, end = a.chunks - 1;
  const int64_t first = k.b * a.seq * heads + k.hv * a.v_dim;
  const auto ahead_of = [](int64_t c) { return c > 0 ? c - 1 : 0; };
  if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 8)) {
    const TileRows<const T> from(a.d_o + first, heads, k.w, k.g, k.col(0));
    bf16x8 pf[2][kPieces], qf[MT][2][NP];
    T raw[4];
    RowGates at;
    // dO of a chunk, and e dO, to LDS.
    const auto put = [&](int64_t c) {
      floatx4 v, x;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = k.tile_value(raw, c, 0, r);
        x[r] = at.doc[r] == 0.f ? v[r] * (a.scale * at.e[r]) : 0.f;
      }
      put_tile<NP>(s.d_o[0][0], k.w, v);
      put_tile<kPieces>(s.u[0], k.w, x);
      if (at.first != at.last) k.mark(s.xs[1][0], s.bad[1][0], v);
    };
    const auto make_z = [&](int64_t c) {
      floatx4 z;
      if (at.first == at.last || !tri_apart<true>(s.bad[1][0], s.xs[1][0], k.tri + (2 * c + 1) * K::kTriPart,
                                                  k.vec + c * 4 * kC + 3 * kC, k.w, z))
        z = tri_product<NP>(pf, s.d_o[0][0]);
      beside.z[k.w][k.lane] = z;
    };
    at.load(k.vec + end * 4 * kC, k.w, k.g);
    from.load(k, end, 0, raw);
    load_tri<true>(k.tri + (2 * end + 1) * K::kTriPart, a.zeros, k.w, pf);
    k.load_cols(end, 2, qf);
    put(end);
    lds_barrier();
    make_z(end);
    for (int64_t c = end; c >= 0; --c) {
      const int64_t ahead = ahead_of(c);
      from.load(k, ahead, 0, raw);
      load_tri<true>(k.tri + (2 * ahead + 1) * K::kTriPart, a.zeros, k.w, pf);
      if (at.last != 0.f) k.cut_cols(qf, k.vec + c * 4 * kC + 3 * kC, 0.f);
      lds_barrier();
      at.load(k.vec + ahead * 4 * kC, k.w, k.g);
      floatx4 S[MT] = {};
      k.col_product(qf, s.u[0], S);
#pragma unroll
      for (int t = 0; t < MT; ++t) beside.s[t][k.w][k.lane] = S[t];
      k.load_cols(ahead, 2, qf);
      lds_barrier();
      put(ahead);
      lds_barrier();
      make_z(ahead);
    }
    return;
  }
  const TileRows<T> to(a.dv + first, heads, k.w, k.g, k.col(0));
  floatx4 S[MT];  // the gradient of the state after the chunk
  k.load_state(a.dh_last, 0, S);
  k.put_state(s.state[end & 1][0], S);
  bf16x8 kf[KS][NP], tf[2][kPieces], cf[MT][2][NP];
  RowGates next;
  next.load(k.vec + end * 4 * kC, k.w, k.g);
  k.load_rows(end, 0, kf);
  load_tri<true>(k.tri + 2 * end * K::kTriPart, a.zeros, k.w, tf);
  k.load_cols(end, 1, cf);
  lds_barrier();
  for (int64_t c = end; c >= 0; --c) {
    const int64_t ahead = ahead_of(c);
    const RowGates at = next;
    const float* doc = k.vec + c * 4 * kC + 3 * kC;
    const bool mixed = at.first != at.last, cut = at.last != 0.f;
    if (cut) k.cut_cols(cf, doc, 0.f);
    lds_barrier();
    next.load(k.vec + ahead * 4 * kC, k.w, k.g);
    const floatx4 ks = k.row_product(kf, s.state[c & 1][0]);
    k.load_rows(ahead, 0, kf);
    floatx4 z = beside.z[k.w][k.lane], y, v;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      z[r] *= a.scale;
      if (at.doc[r] == at.last) z[r] = fmaf(at.end[r], ks[r], z[r]);
    }
    put_tile<kPieces>(s.x[0], k.w, z);
    if (mixed) k.mark(s.xs[0][0], s.bad[0][0], z);
    lds_barrier();
    k.store_padded(a.dstates, c, 0, S);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const floatx4 q = beside.s[t][k.w][k.lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) S[t][r] = cut ? q[r] : fmaf(S[t][r], at.all, q[r]);
    }
    if (!mixed || !tri_apart<true>(s.bad[0][0], s.xs[0][0], k.tri + 2 * c * K::kTriPart, doc, k.w, z))
      z = tri_product<kPieces>(tf, s.x[0]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      y[r] = at.beta[r] * z[r];
      v[r] = at.doc[r] == 0.f ? -y[r] * at.e[r] : 0.f;
    }
    put_tile<kPieces>(s.y[0], k.w, v);
    load_tri<true>(k.tri + 2 * ahead * K::kTriPart, a.zeros, k.w, tf);
    lds_barrier();
    k.col_product(cf, s.y[0], S);
    k.put_state(s.state[(c + 1) & 1][0], S);
    k.load_cols(ahead, 1, cf);
    k.store_rows(a.z, c, 0, z);
    to.store(k, c, 0, y);
  }
  if (a.dh0 && k.holds) k.store_state(a.dh0, 0, S);
}

// ---------------------------------------------------------------------------
// The gradients of q, k, g and beta: a chunk of a value head to a workgroup of four waves, wave w the
// columns 16 w.. of everything turned (tokens as columns). Operands pass through LDS 32 columns of v_dim
// at a time, as fragments with their columns in order. 1536 chunks of 128 by 128 in 203 us, 500 MB at
// 2.5 TB/s: what is loaded is cut into pieces by the lanes that load it, and all waits for that.
// ---------------------------------------------------------------------------
// Of wide keys four waves have the same columns and a quarter of k_dim each: with the gradients of q and k
// in the registers of one, a SIMD had room for two waves, which could not hide what they wait for.
template <int KD>
constexpr int kGradParts = KD > 64 ? 4 : 1;

template <typename T, int KD>
struct GradShared {
  union {
    struct {
      uint16_t u[4 * kPieces * kFrag], z[4 * kPieces * kFrag], d_o[4 * kIn<T> * kFrag];
      uint16_t S[KD / 16 * kPieces * kFrag], dS[KD / 16 * kPieces * kFrag];
    };
    // Then, of several parts, D dP and M of each wave's columns: the one or two fragments of what its
    // tokens read and those of what reads them, three in all.
    uint16_t tokens[kGradParts<KD> > 1 ? 2 : 1][kGradParts<KD> > 1 ? 4 : 1][3 * kPieces * kFrag];
  };
  double G[kC];
  float beta[kC], into[kGradParts<KD>][kC], w[kGradParts<KD>][kC], dbeta[kC], dot[16];
  float across[kGradParts<KD> > 1 ? 2 : 1][4][kC];  // sums of W over j < t <= i, i of a wave
  floatx4 dots[2][kGradParts<KD> > 1 ? 10 : 1][64];  // of several parts: q's and k's dot products with earlier keys
  int doc[kC];
};

// Eight values of row `row`, columns 8 c.., into fragments of N pieces.
template <int N>
__device__ inline void stage(uint16_t* to, int row, int c, float (&x)[8]) {
  bf16x8 p[N];
  split<N>(x, p);
  store_frag(to + row / 16 * N * kFrag, c * 16 + (row & 15), p);
}

template <typename T, int KD>
__global__ __launch_bounds__(256 * kGradParts<KD>, kGradParts<KD> > 1 ? 4 : 2) void delta_grad_kernel(Args<T> a) {
  constexpr int NP = kIn<T>, H = kGradParts<KD>, MT = KD / 16 / H, kPart = KD / 8 * NP * kFrag;
  __shared__ __attribute__((aligned(16))) GradShared<T, KD> s;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, m = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = wave & 3, part = wave >> 2;
  const int64_t unit = xcd_order(blockIdx.x, gridDim.x), chunk = unit % a.chunks, bh = unit / a.chunks;
  const int64_t b = bh / a.v_heads, hv = bh % a.v_heads, hk = hv / (a.v_heads / a.k_heads);
  const int64_t t0 = chunk * kC;
  // What this thread stages: a row of the states (parts 0 and 1), of u and z (part 2), of dO (part 3).
  const int row = tid >> 2, c8 = tid & 3, token = row & 63;
  const uint32_t at_token = token * a.v_pad + 8 * c8, at_row = row * a.v_pad + 8 * c8;
  const float *resid = a.resid + unit * kC * a.v_pad, *zs = a.z + unit * kC * a.v_pad;
  const float *st = a.states + unit * KD * a.v_pad, *ds = a.dstates + unit * KD * a.v_pad;
  float dot_b = 0.f, dot_s = 0.f;

  // The wave's column is token `mine`.
  const int mine = 16 * w + m;
  const int64_t t = t0 + mine;
  const bool here = t < a.seq;
  const T* qrow = a.q + b * a.q_b + (here ? t : a.seq - 1) * a.q_t + hk * a.q_h;
  const T* krow = a.k + b * a.k_b + (here ? t : a.seq - 1) * a.k_t + hk * a.k_h;
  const uint16_t* kr = a.keys + ((b * a.k_heads + hk) * a.chunks + chunk) * (3 * kPart);
  // The dot products of the wave's tokens' q and k with the keys of tokens 16 n.. Where k_dim is a multiple of
  // four, what lies past it is loaded from within and cut, so that loads are under way together (behind a test
  // of where the row ends each waits for the one before: 222 us for 205).
  const auto keys_dots = [&](int n, floatx4& q_dots, floatx4& k_dots) {
    q_dots = k_dots = (floatx4){};
    const auto sum = [&](const auto& row_of_q) {
#pragma unroll
      for (int i = 0; i < KD / 32; ++i) {
        float x[8];
        bf16x8 f[NP], own[NP], kn[NP];
        row_of_q(i, x);
        split<NP>(x, f);
        load_frag(kr + (w * (KD / 32) + i) * NP * kFrag, lane, own);
        load_frag(kr + (n * (KD / 32) + i) * NP * kFrag, lane, kn);
        q_dots = mma(kn, f, q_dots);
        k_dots = mma(kn, own, k_dots);
      }
      q_dots = settled(q_dots), k_dots = settled(k_dots);
    };
    if (a.k_dim % 4 == 0) {
      sum([&](int i, float (&x)[8]) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int at = 32 * i + 16 * half + 4 * g;
          const bool in = here && at < a.k_dim;
          float v[4];
          load_part(qrow, in ? at : 0, 4, v);
#pragma unroll
          for (int c = 0; c < 4; ++c) x[4 * half + c] = in ? v[c] : 0.f;
        }
      });
    } else sum([&](int i, float (&x)[8]) { load_row8(qrow, i, g, here ? a.k_dim : 0, x); });
  };
  if (wave == (H > 1 ? 4 : 0)) {  // (the second part's first wave has no dot products)
    const Gates x = chunk_gates(a, b, hv, t0);
    s.G[lane] = x.G;
    s.beta[lane] = x.beta;
    s.doc[lane] = x.doc;
  }
  if constexpr (H > 1) {  // a part the keys 16 part..
    if (part <= w) {
      const int at = w * (w + 1) / 2 + part;
      floatx4 q_dots, k_dots;
      keys_dots(part, q_dots, k_dots);
      s.dots[0][at][lane] = q_dots, s.dots[1][at][lane] = k_dots;
    }
  }

  // Slot n of the first w + 1: rows of u (tokens 16 n..) against the wave's columns of dO and of z; slot
  // n + 1 of the others: rows of dO and of z against its columns of u. (Of several parts the first takes
  // dO and the second z, both in p.)
  floatx4 p[5] = {}, mm[H == 1 ? 5 : 1] = {}, dq[MT] = {}, ka[MT] = {}, kb[MT] = {};
  for (int v0 = 0; v0 < a.v_pad; v0 += 32) {
    __syncthreads();
    float x[8], y[8];
    if (H == 1 || part == 2) {
      load_vec<float, 8>(resid + (at_token + v0), x);
      load_vec<float, 8>(zs + (at_token + v0), y);
      const float beta = s.beta[token];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dot_b = fmaf(x[i], y[i], dot_b);
        x[i] *= beta;
      }
      stage<kPieces>(s.u, token, c8, x);
      stage<kPieces>(s.z, token, c8, y);
    }
    if (H == 1 || part == 3) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = v0 + 8 * c8 + 4 * h;
        float q[4] = {0.f, 0.f, 0.f, 0.f};
        if (t0 + token < a.seq && at < a.v_dim)
          load_part(a.d_o + ((b * a.seq + t0 + token) * a.v_heads + hv) * a.v_dim, at, a.v_dim - at, q);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * h + i] = q[i];
      }
      stage<NP>(s.d_o, token, c8, x);
    }
    if (row < KD) {
      load_vec<float, 8>(st + (at_row + v0), x);
      load_vec<float, 8>(ds + (at_row + v0), y);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot_s = fmaf(x[i], y[i], dot_s);
      stage<kPieces>(s.S, row, c8, x);
      stage<kPieces>(s.dS, row, c8, y);
    }
    __syncthreads();
    bf16x8 uw[kPieces], zw[kPieces], ow[NP];
    load_frag(s.u + w * kPieces * kFrag, lane, uw);
    load_frag(s.z + w * kPieces * kFrag, lane, zw);
    load_frag(s.d_o + w * NP * kFrag, lane, ow);
#pragma unroll
    for (int n = 0; n < 5; ++n) {
      if (n <= w) {
        bf16x8 un[kPieces];
        load_frag(s.u + n * kPieces * kFrag, lane, un);
        if (part == 0) p[n] = mma(un, ow, p[n]);
        if constexpr (H == 1) mm[n] = mma(un, zw, mm[n]);
        else if (part == 1) p[n] = mma(un, zw, p[n]);
      } else {
        if (part == 0) {
          bf16x8 on[NP];
          load_frag(s.d_o + (n - 1) * NP * kFrag, lane, on);
          p[n] = mma(on, uw, p[n]);
        }
        if (H == 1 || part == 1) {
          bf16x8 zn[kPieces];
          load_frag(s.z + (n - 1) * kPieces * kFrag, lane, zn);
          if constexpr (H == 1) mm[n] = mma(zn, uw, mm[n]);
          else p[n] = mma(zn, uw, p[n]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int tile = part * MT + i;
      bf16x8 f[kPieces];
      load_frag(s.S + tile * kPieces * kFrag, lane, f);
      dq[i] = mma(f, ow, dq[i]);
      ka[i] = mma(f, zw, ka[i]);
      load_frag(s.dS + tile * kPieces * kFrag, lane, f);
      kb[i] = mma(f, uw, kb[i]);
    }
  }

  const int doc = s.doc[mine], last = s.doc[kC - 1];
  const double Gm = s.G[mine];
  const float bm = s.beta[mine];
  const float e = doc == 0 ? expf((float)Gm) : 0.f;
  const float et = doc == last ? expf((float)(s.G[kC - 1] - Gm)) : 0.f;
  float wrote = 0.f, into = 0.f;  // k . (dS' u), and what the state's decay up to the token passes on
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    dq[i] = settled(dq[i]), ka[i] = settled(ka[i]), kb[i] = settled(kb[i]);
    const int d = 16 * (part * MT + i) + 4 * g;
    float qv[4] = {0.f, 0.f, 0.f, 0.f}, kv[4] = {0.f, 0.f, 0.f, 0.f};
    if (here && d < a.k_dim) {
      load_part(qrow, d, a.k_dim - d, qv);
      load_part(krow, d, a.k_dim - d, kv);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      dq[i][r] = doc == 0 ? dq[i][r] * (a.scale * e) : 0.f;
      ka[i][r] = doc == 0 ? ka[i][r] * (-e * bm) : 0.f;
      kb[i][r] = doc == last ? kb[i][r] * et : 0.f;
      into = fmaf(qv[r], dq[i][r], into);
      into = fmaf(kv[r], ka[i][r], into);
      wrote = fmaf(kv[r], kb[i][r], wrote);
    }
  }
  into += __shfl_xor(into, 16);
  into += __shfl_xor(into, 32);
  wrote += __shfl_xor(wrote, 16);
  wrote += __shfl_xor(wrote, 32);
  if (g == 0) {
    s.into[part][mine] = into;
    s.w[part][mine] = wrote;
  }
  // D dP (turned in the first w + 1 slots), and M.
  if (H == 1 || part < 2) {
#pragma unroll
    for (int n = 0; n < 5; ++n) {
      const bool turned = n <= w;
      const int first = 16 * (turned ? n : n - 1) + 4 * g, way = turned ? 1 : -1;
      p[n] = settled(p[n]);
      if constexpr (H == 1) mm[n] = settled(mm[n]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int other = first + r, apart = (mine - other) * way;
        const bool one = (s.doc[other] == doc) & (apart >= 0);
        const float gap = (float)((Gm - s.G[other]) * way);
        const float D = expf(one ? gap : -1e4f);  // else 0
        const float bi = turned ? bm : s.beta[other], below = apart ? -bi * D : 0.f;
        if constexpr (H == 1) {
          p[n][r] = one ? p[n][r] * (D * a.scale) : 0.f;
          mm[n][r] = one && apart ? mm[n][r] * below : 0.f;
        } else {
          const float by = part == 0 ? D * a.scale : below;
          p[n][r] = one && (part == 0 || apart) ? p[n][r] * by : 0.f;
        }
      }
    }
  }
  // Sums of W over j < t, and over the wave's i >= t.
  if (H == 1 || part < 2) {
    floatx4 W[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      W[n] = (floatx4){};
      if (n > w) continue;
      if constexpr (H == 1) {
        floatx4 q_dots, k_dots;
        keys_dots(n, q_dots, k_dots);
        W[n] = p[n] * q_dots + mm[n] * k_dots;
      } else {
        W[n] = p[n] * s.dots[part][w * (w + 1) / 2 + n][lane];
      }
    }
    float before = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const float s0 = W[n][0], s1 = s0 + W[n][1], s2 = s1 + W[n][2];
      float sum = s2 + W[n][3];
      float other = __shfl_up(sum, 16);
      if (g >= 1) sum += other;
      other = __shfl_up(sum, 32);
      if (g >= 2) sum += other;
      other = __shfl_up(sum, 16);
      const float left = g ? before + other : before;
      before += __shfl(sum, 48 + m);
      floatx4 y = {left, left + s0, left + s1, left + s2};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (16 * n + 4 * g + r > mine) y[r] = 0.f;
        y[r] += lane_xor1(y[r]);
        y[r] += lane_xor2(y[r]);
        y[r] += row_rot4(y[r]);
        y[r] += row_rot8(y[r]);
      }
      if (m == 0) *reinterpret_cast<floatx4*>(&s.across[H == 1 ? 0 : part][w][16 * n + 4 * g]) = y;
    }
  }
  const floatx4 none = {};
  // The slots as right operands: columns that the wave's tokens read (ks of the first two), and that read
  // them.
  const auto reads = [&](const floatx4 (&v)[5], int ks, bf16x8 (&f)[kPieces]) {
    split<kPieces>(v[2 * ks], 2 * ks + 1 <= w ? v[2 * ks + 1] : none, f);
  };
  const auto read_by = [&](const floatx4 (&v)[5], int ks, bf16x8 (&f)[kPieces]) {
    split<kPieces>(2 * ks >= w ? v[2 * ks + 1] : none, v[2 * ks + 2], f);
  };
  if constexpr (H > 1) {
    __syncthreads();
    uint16_t* to = s.tokens[part & 1][w];
    bf16x8 f[kPieces];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (part > 1) break;
      // In their order: ks of what is read, then of what reads.
      if (2 * ks <= w) {
        reads(p, ks, f);
        store_frag(to + ks * kPieces * kFrag, lane, f);
      }
      if (2 * ks + 1 >= w) {
        read_by(p, ks, f);
        store_frag(to + (w < 2 ? 1 + ks : 2) * kPieces * kFrag, lane, f);
      }
    }
    __syncthreads();
  }
  const uint16_t* kt = kr + kPart + part * MT * 2 * NP * kFrag;
  const uint16_t* qt = kt + kPart;
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    if (2 * ks <= w) {
      bf16x8 pf[kPieces], mf[kPieces];
      if constexpr (H == 1) {
        reads(p, ks, pf);
        reads(mm, ks, mf);
      } else {
        load_frag(s.tokens[0][w] + ks * kPieces * kFrag, lane, pf);
        load_frag(s.tokens[1][w] + ks * kPieces * kFrag, lane, mf);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        bf16x8 f[NP];
        load_frag(kt + (i * 2 + ks) * NP * kFrag, lane, f);
        dq[i] = mma(f, pf, dq[i]);
        ka[i] = mma(f, mf, ka[i]);
      }
    }
    if (2 * ks + 1 >= w) {
      bf16x8 pf[kPieces], mf[kPieces];
      if constexpr (H == 1) {
        read_by(p, ks, pf);
        read_by(mm, ks, mf);
      } else {
        const int at = (w < 2 ? 1 + ks : 2) * kPieces * kFrag;
        load_frag(s.tokens[0][w] + at, lane, pf);
        load_frag(s.tokens[1][w] + at, lane, mf);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        bf16x8 f[NP];
        load_frag(qt + (i * 2 + ks) * NP * kFrag, lane, f);
        kb[i] = mma(f, pf, kb[i]);
        load_frag(kt + (i * 2 + ks) * NP * kFrag, lane, f);
        kb[i] = mma(f, mf, kb[i]);
      }
    }
  }
  const bool shared = a.k_heads != a.v_heads;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int d = 16 * (part * MT + i) + 4 * g;
    dq[i] = settled(dq[i]), ka[i] = settled(ka[i]), kb[i] = settled(kb[i]);
    if (!here || d >= a.k_dim) continue;
    float dk[4], dqv[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      dk[r] = ka[i][r] + kb[i][r];
      dqv[r] = dq[i][r];
    }
    if (shared) {
      const int64_t at = ((b * a.seq + t) * a.v_heads + hv) * a.k_dim;
      store_part(a.dq_part + at, d, a.k_dim - d, dqv);
      store_part(a.dk_part + at, d, a.k_dim - d, dk);
    } else {
      const int64_t at = ((b * a.seq + t) * a.k_heads + hk) * a.k_dim;
      store_part(a.dq + at, d, a.k_dim - d, dqv);
      store_part(a.dk + at, d, a.k_dim - d, dk);
    }
  }
  dot_b += lane_xor1(dot_b);
  dot_b += lane_xor2(dot_b);
  if (c8 == 0 && part == (H == 1 ? 0 : 2)) s.dbeta[token] = dot_b;
  dot_s = wave_sum_all(dot_s);
  if (lane == 0) s.dot[wave] = dot_s;
  __syncthreads();
  if (wave == 0) {
    const int d = s.doc[lane];
    double v = 0.0, from = 0.0, upto = 0.0;  // W's sums; sums over i >= t, j < t
    float all = 0.f;
#pragma unroll
    for (int n = 0; n < H; ++n) {
      if (d == 0) from += s.into[n][lane];
      if (d == last) upto += s.w[n][lane];
    }
#pragma unroll
    for (int n = 0; n < 4 * H; ++n) all += s.dot[n];
#pragma unroll
    for (int n = 0; n < 4; ++n)
      v += H == 1 ? s.across[0][n][lane] : s.across[0][n][lane] + s.across[H > 1][n][lane];
#pragma unroll
    for (int n = 1; n < 64; n *= 2) {
      const double after = __shfl_down(from, n), before = __shfl_up(upto, n);
      if (lane + n < 64) from += after;
      if (lane >= n) upto += before;
    }
    upto = __shfl_up(upto, 1);
    if (d == 0) v += from;
    if (d == last && lane > 0) v += upto;
    if (last == 0) v += expf((float)s.G[kC - 1]) * all;
    // Nothing decays into a document's first token.
    const int before = __shfl_up(d, 1);
    if (d != (lane == 0 ? 0 : before)) v = 0.0;
    const int64_t to = (b * a.seq + t0 + lane) * a.v_heads + hv;
    if (t0 + lane < a.seq) {
      store_any(a.dg, to, a.g_type, (float)v);
      store_any(a.dbeta, to, a.beta_type, s.dbeta[lane]);
    }
  }
}

// Gradients of q and k that several value heads share: their parts' sum, in the heads' order.
template <typename T>
__global__ __launch_bounds__(256) void delta_share_kernel(Args<T> a) {
  const int64_t n = a.batch * a.seq * a.k_heads * a.k_dim;
  const int group = (int)(a.v_heads / a.k_heads);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t head = i / a.k_dim, at = head * group * a.k_dim + i % a.k_dim;
    float q = 0.f, k = 0.f;
    for (int j = 0; j < group; ++j) {
      q += a.dq_part[at + (int64_t)j * a.k_dim];
      k += a.dk_part[at + (int64_t)j * a.k_dim];
    }
    store_scalar(a.dq + i, q);
    store_scalar(a.dk + i, k);
  }
}

// ---------------------------------------------------------------------------
// One token of each sequence: the state is read and written once, a workgroup 64 columns of a head; lane
// l of wave w has columns 4 (l % 16).. of rows l / 16 + 4 w + 16 n. 192 states of 128 by 128 (25 MB) take
// 8.6 us, of which a launch alone takes 2.4: one load's wait, the sums over the rows and the store one after
// another.
// ---------------------------------------------------------------------------
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void delta_step_kernel(Args<T> a, float* h) {
  __shared__ __attribute__((aligned(16))) float red[2][4][64];
  const int tid = threadIdx.x, c4 = (tid & 15) * 4, r0 = tid >> 4;
  const int tiles = (a.v_dim + 63) / 64;
  const int64_t unit = blockIdx.x, bh = unit / tiles;
  const int64_t b = bh / a.v_heads, hv = bh % a.v_heads, hk = hv / (a.v_heads / a.k_heads);
  const int col = (int)(unit % tiles) * 64 + c4, left = a.v_dim - col;
  const T* q = a.q + b * a.q_b + hk * a.q_h;
  const T* k = a.k + b * a.k_b + hk * a.k_h;
  float* at = h + bh * a.k_dim * a.v_dim;
  const float decay = expf(load_any(a.g, bh, a.g_type)), beta = load_any(a.beta, bh, a.beta_type);
  float S[ROWS][4], kr[ROWS], x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
  float v[4] = {0.f, 0.f, 0.f, 0.f}, qk = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c < left) v[c] = load_scalar(a.v + b * a.v_b + hv * a.v_h + col + c);
#pragma unroll
  for (int n = 0; n < ROWS; ++n) {
    const int d = r0 + 16 * n;
    const bool in = d < a.k_dim;
    kr[n] = in ? load_scalar(k + d) : 0.f;
    const float qr = in ? load_scalar(q + d) : 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) S[n][c] = 0.f;
    if (in && left > 0) load_part(at, (uint32_t)(d * a.v_dim + col), left, S[n]);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      S[n][c] *= decay;
      x[c] = fmaf(kr[n], S[n][c], x[c]);
      y[c] = fmaf(qr, S[n][c], y[c]);
    }
    qk = fmaf(qr, kr[n], qk);
  }
  // o = S_t^T q = p^T q + (q . k) beta r: all sums over the old state in one pass.
  __shared__ float dots[4];
  qk += __shfl_xor(qk, 16);
  qk += __shfl_xor(qk, 32);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    x[c] += __shfl_xor(x[c], 16);
    x[c] += __shfl_xor(x[c], 32);
    y[c] += __shfl_xor(y[c], 16);
    y[c] += __shfl_xor(y[c], 32);
  }
  if ((tid & 63) < 16) {
    *(floatx4*)&red[0][tid >> 6][c4] = floatx4{x[0], x[1], x[2], x[3]};
    *(floatx4*)&red[1][tid >> 6][c4] = floatx4{y[0], y[1], y[2], y[3]};
    if (c4 == 0) dots[tid >> 6] = qk;
  }
  __syncthreads();
  qk = (dots[0] + dots[1]) + (dots[2] + dots[3]);
  float wr[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    x[c] = y[c] = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      x[c] += red[0][n][c4 + c];
      y[c] += red[1][n][c4 + c];
    }
    wr[c] = beta * (v[c] - x[c]);
    y[c] = a.scale * fmaf(qk, wr[c], y[c]);
  }
#pragma unroll
  for (int n = 0; n < ROWS; ++n) {
    const int d = r0 + 16 * n;
#pragma unroll
    for (int c = 0; c < 4; ++c) S[n][c] = fmaf(kr[n], wr[c], S[n][c]);
    if (d < a.k_dim && left > 0) store_part(at, (uint32_t)(d * a.v_dim + col), left, S[n]);
  }
  if (r0 == 0 && left > 0) store_part(a.o + bh * a.v_dim, (uint32_t)col, left, y);
}

// Launches by type and k_dim.
template <typename T>
int launch_fwd(const Args<T>& a, hipStream_t s);
template <typename T>
int launch_bwd(const Args<T>& a, hipStream_t s);
template <typename T>
int launch_step(const Args<T>& a, float* h, hipStream_t s);

}  // namespace delta
}  // namespace mqc
