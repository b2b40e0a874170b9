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
//   dG_i = q_i . dQ_i + k_i . (the first bracket - the second), dG_63 also the second bracket's last part
//   and e_63 <dS', S>; dg_t is the sum of dG from t to its document's end.
//
// Three kinds of kernels. One over all chunks side by side forms the products within them (gram
// matrices, the triangular inverse) and lays every operand out as the matrix instructions read it. One
// walks the chunks of a head: columns of S do not depend on one another, so each wave owns 16 of them and
// keeps them in registers from the first chunk to the last, with no barrier and no word to another wave:
// what a product leaves (a column a lane, four rows each) is what the next one takes as its right operand
// if the left one's columns are in the order kPlace. The backward's gradients of q, k, g and beta need
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
  uint16_t *keys, *tri;
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
// that share it; wave w rows 16 w.
// ---------------------------------------------------------------------------
template <typename T, int KD, bool BWD>
struct PrepShared {
  uint16_t frags[KD / 8 * kIn<T> * kFrag];  // K by rows; then Q, to be turned
  float kk[kC][kC + 1], qk[kC][kC + 1];     // below the diagonal and on it
  float m[kC][kC + 1], inv[kC][kC + 1], y[3][16][17];
  double G[kC];
  float beta[kC];
  int doc[kC];
};

// X = (I + m)^-1 for a strictly lower triangular m, rows by substitution in blocks of 16, then block
// diagonal by block diagonal: X_ij = -X_ii (sum over j <= l < i of m_il X_lj).
template <typename S>
__device__ inline void invert(S& s) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, o = 16 * w;
  if (lane < 16) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == lane ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j < i) v = fmaf(-s.m[o + i][o + j], x[j], v);
      x[i] = i < lane ? 0.f : v;
      s.inv[o + i][o + lane] = x[i];
    }
  }
  const int r = tid >> 4, c = tid & 15;
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    __syncthreads();
    for (int b = 0; b + d < 4; ++b) {
      const int i = 16 * (b + d), j = 16 * b;
      float v = 0.f;
      for (int l = j; l < i; ++l) v = fmaf(s.m[i + r][l], s.inv[l][j + c], v);
      s.y[b][r][c] = v;
    }
    __syncthreads();
    for (int b = 0; b + d < 4; ++b) {
      const int i = 16 * (b + d), j = 16 * b;
      float v = 0.f;
#pragma unroll
      for (int l = 0; l < 16; ++l) v = fmaf(-s.inv[i + r][i + l], s.y[b][l][c], v);
      s.inv[i + r][j + c] = v;
    }
  }
  __syncthreads();
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
  __shared__ __attribute__((aligned(16))) PrepShared<T, KD, BWD> s;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, m = lane & 15;
  const int64_t unit = blockIdx.x, chunk = unit % a.chunks, bh = unit / a.chunks;
  const int64_t b = bh / a.k_heads, hk = bh % a.k_heads, t0 = chunk * kC, t = t0 + 16 * w + m;
  const int group = (int)(a.v_heads / a.k_heads);
  uint16_t* keys = a.keys + unit * (3 * KD / 8 * NP * kFrag);
  constexpr int kPart = KD / 8 * NP * kFrag;

  // Rows of K and Q as fragments.
  bf16x8 kf[KS][NP], qf[KS][NP];
  {
    const T* krow = a.k + b * a.k_b + t * a.k_t + hk * a.k_h;
    const T* qrow = a.q + b * a.q_b + t * a.q_t + hk * a.q_h;
    const int dim = t < a.seq ? a.k_dim : 0;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      float x[8];
      load_row8(krow, i, g, dim, x);
      split<NP>(x, kf[i]);
      load_row8(qrow, i, g, dim, x);
      split<NP>(x, qf[i]);
      const int at = (i * 4 + w) * NP * kFrag;
      store_frag(keys + at, lane, kf[i]);
      store_frag(s.frags + at, lane, kf[i]);
      if constexpr (!BWD) store_frag(keys + 2 * kPart + at, lane, qf[i]);
    }
  }
  __syncthreads();
  for (int n = 0; n <= w; ++n) {
    floatx4 kk = {}, qk = {};
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      bf16x8 kn[NP];
      load_frag(s.frags + (i * 4 + n) * NP * kFrag, lane, kn);
      kk = mma(kf[i], kn, kk);
      qk = mma(qf[i], kn, qk);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s.kk[16 * w + 4 * g + r][16 * n + m] = kk[r];
      s.qk[16 * w + 4 * g + r][16 * n + m] = qk[r];
    }
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
    __syncthreads();  // the head before is done with what follows
    if (w == 0) {
      const Gates x = chunk_gates(a, b, hv, t0);
      s.G[lane] = x.G;
      s.beta[lane] = x.beta;
      s.doc[lane] = x.doc;
      const double end = __shfl(x.G, 63);
      float* vec = a.vec + at * 4 * kC;
      vec[lane] = x.doc == 0 ? expf((float)x.G) : 0.f;
      vec[kC + lane] = x.doc == __shfl(x.doc, 63) ? expf((float)(end - x.G)) : 0.f;
      vec[2 * kC + lane] = x.beta;
      vec[3 * kC + lane] = (float)x.doc;
    }
    __syncthreads();
    // m and P (over m's and qk's places above the diagonal nothing is read but as zero).
    float P[kC * kC / 256];
    for (int i = 0; i < kC * kC / 256; ++i) {
      const int row = i * 4 + w, col = lane;
      const bool seen = col <= row && s.doc[row] == s.doc[col];
      const float D = seen ? expf((float)(s.G[row] - s.G[col])) : 0.f;
      s.m[row][col] = seen && col < row ? D * s.kk[row][col] * s.beta[BWD ? row : col] : 0.f;
      P[i] = seen ? D * s.qk[row][col] : 0.f;
      s.inv[row][col] = 0.f;
    }
    __syncthreads();
    invert(s);
    for (int i = 0; i < kC * kC / 256; ++i) s.m[i * 4 + w][lane] = P[i];
    __syncthreads();
    uint16_t* tri = a.tri + at * (2 * kTri * kPieces * kFrag);
    for (int f = w; f < 2 * kTri; f += 4) {
      const int n = f % kTri;  // which rows of 16 and columns of 32
      const int mt = BWD ? (n < 4 ? n / 2 : n - 2) : (n < 2 ? n : n / 2 + 1);
      const int ks = BWD ? (n < 4 ? n % 2 : 1) : (n < 2 ? 0 : n % 2);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = 16 * mt + m, col = 32 * ks + place(g, e);
        const int i = BWD ? col : row, l = BWD ? row : col;
        // Not of another document (whose NaN may have come here) and not above the diagonal.
        x[e] = l > i || s.doc[i] != s.doc[l] ? 0.f : f < kTri ? s.inv[i][l] : s.m[i][l];
      }
      bf16x8 p[kPieces];
      split<kPieces>(x, p);
      store_frag(tri + f * kPieces * kFrag, lane, p);
    }
  }
}

// ---------------------------------------------------------------------------
// The walks. A wave has 16 columns of a head's state.
// ---------------------------------------------------------------------------

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
__device__ inline bool finite(const floatx4 (&x)[4]) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) ok = ok && finite(x[i][r]);
  return __ballot(!ok) == 0;
}

// tri x, a triangular matrix [64, 64] (its fragments) times the wave's columns. Where documents meet in
// the chunk (`mixed`) and x is not finite, term by term: zero times NaN is not zero.
template <bool UPPER>
__device__ inline void tri_product(const uint16_t* tri, const floatx4 (&x)[4], bool mixed,
                                   const float* doc, float (*xs)[17], floatx4 (&out)[4]) {
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  if (mixed && !finite(x)) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) xs[16 * i + 4 * g + r][m] = x[i][r];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * i + 4 * g + r;
        float v = 0.f;
        for (int j = UPPER ? row : 0; UPPER ? j < kC : j <= row; ++j)
          if (doc[j] == doc[row]) v = fmaf(tri_at<UPPER>(tri, row, j), xs[j][m], v);
        out[i][r] = v;
      }
    __syncthreads();
    return;
  }
  bf16x8 xf[2][kPieces];
#pragma unroll
  for (int s = 0; s < 2; ++s) split<kPieces>(x[2 * s], x[2 * s + 1], xf[s]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    floatx4 v = {};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int f = UPPER ? upper_frag(i, s) : lower_frag(i, s);
      if (f < 0) continue;
      bf16x8 tf[kPieces];
      load_frag(tri + f * kPieces * kFrag, lane, tf);
      v = mma(tf, xf[s], v);
    }
    out[i] = v;
  }
}

// rows x S for the chunk's rows (K or Q as fragments by rows) and the state's pieces.
template <int KS, int NP>
__device__ inline void row_product(const uint16_t* rows, const bf16x8 (&sf)[KS][kPieces],
                                   floatx4 (&out)[4]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    floatx4 v = {};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      bf16x8 f[NP];
      load_frag(rows + (s * 4 + i) * NP * kFrag, lane, f);
      v = mma(f, sf[s], v);
    }
    out[i] = v;
  }
}

// S += cols x for K^T or Q^T as fragments; tokens of other documents than `keep` left out where `cut`.
template <int KD, int NP>
__device__ inline void col_product(const uint16_t* cols, const floatx4 (&x)[4], bool cut,
                                   const float* doc, float keep, floatx4 (&S)[KD / 16]) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  bf16x8 xf[2][kPieces];
#pragma unroll
  for (int s = 0; s < 2; ++s) split<kPieces>(x[2 * s], x[2 * s + 1], xf[s]);
  if (cut) {
    u32x4 mask[2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t e = doc[32 * s + place(g, j)] == keep ? 0xffffu : 0u;
        mask[s][j / 2] = j % 2 ? mask[s][j / 2] | e << 16 : e;
      }
#pragma unroll
    for (int i = 0; i < KD / 16; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bf16x8 f[NP];
        load_frag(cols + (i * 2 + s) * NP * kFrag, lane, f);
#pragma unroll
        for (int p = 0; p < NP; ++p)
          f[p] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, f[p]) & mask[s]);
        S[i] = mma(f, xf[s], S[i]);
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < KD / 16; ++i)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 f[NP];
      load_frag(cols + (i * 2 + s) * NP * kFrag, lane, f);
      S[i] = mma(f, xf[s], S[i]);
    }
}

// The wave's columns of a state [k_dim, v_dim] in memory.
template <int KD, typename T>
__device__ inline void load_state(const Args<T>& a, const float* from, int col, floatx4 (&S)[KD / 16]) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < KD / 16; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * i + 4 * g + r;
      S[i][r] = from && d < a.k_dim && col < a.v_dim ? from[(int64_t)d * a.v_dim + col] : 0.f;
    }
}
template <int KD, typename T>
__device__ inline void store_state(const Args<T>& a, float* to, int col, const floatx4 (&S)[KD / 16]) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < KD / 16; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * i + 4 * g + r;
      if (d < a.k_dim && col < a.v_dim) to[(int64_t)d * a.v_dim + col] = S[i][r];
    }
}
// The same between chunks, padded.
template <int KD>
__device__ inline void store_padded(float* to, int64_t pitch, const floatx4 (&S)[KD / 16]) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < KD / 16; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) to[(16 * i + 4 * g + r) * pitch] = S[i][r];
}

template <typename T, int KD>
__global__ __launch_bounds__(64) void delta_fwd_kernel(Args<T> a) {
  constexpr int NP = kIn<T>, KS = KD / 32, kPart = KD / 8 * NP * kFrag;
  __shared__ float xs[kC][17];
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  const int tiles = a.v_pad / 16;
  const int64_t unit = xcd_order(blockIdx.x, gridDim.x), bh = unit / tiles;
  const int64_t b = bh / a.v_heads, hv = bh % a.v_heads, hk = hv / (a.v_heads / a.k_heads);
  const int col = (int)(unit % tiles) * 16 + m;
  const bool real = col < a.v_dim;
  const T* v = a.v + b * a.v_b + hv * a.v_h + col;
  const uint16_t* keys = a.keys + (b * a.k_heads + hk) * a.chunks * (3 * kPart);
  const uint16_t* tri = a.tri + bh * a.chunks * (2 * kTri * kPieces * kFrag);
  const float* vec = a.vec + bh * a.chunks * (4 * kC);
  floatx4 S[KD / 16];
  load_state<KD>(a, a.h0 ? a.h0 + bh * a.k_dim * a.v_dim : nullptr, col, S);
  for (int64_t c = 0; c < a.chunks; ++c) {
    const float* doc = vec + 3 * kC;
    const bool mixed = doc[0] != doc[kC - 1];
    if (a.states) store_padded<KD>(a.states + (bh * a.chunks + c) * KD * a.v_pad + col, a.v_pad, S);
    bf16x8 sf[KS][kPieces];
#pragma unroll
    for (int s = 0; s < KS; ++s) split<kPieces>(S[2 * s], S[2 * s + 1], sf[s]);
    floatx4 x[4], r[4];
    row_product<KS, NP>(keys, sf, x);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 16 * i + 4 * g + j;
        const int64_t t = c * kC + row;
        const float vt = real && t < a.seq ? load_scalar(v + t * a.v_t) : 0.f;
        x[i][j] = doc[row] == 0.f && t < a.seq ? fmaf(-vec[row], x[i][j], vt) : vt;
      }
    tri_product<false>(tri, x, mixed, doc, xs, r);
    if (a.resid) {
      float* to = a.resid + (bh * a.chunks + c) * kC * a.v_pad + col;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) to[(int64_t)(16 * i + 4 * g + j) * a.v_pad] = r[i][j];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) r[i][j] *= vec[2 * kC + 16 * i + 4 * g + j];
    floatx4 y[4];
    row_product<KS, NP>(keys + 2 * kPart, sf, x);
    tri_product<false>(tri + kTri * kPieces * kFrag, r, mixed, doc, xs, y);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 16 * i + 4 * g + j;
        const int64_t t = c * kC + row;
        const float ot = a.scale * (doc[row] == 0.f ? fmaf(vec[row], x[i][j], y[i][j]) : y[i][j]);
        if (real && t < a.seq)
          store_scalar(a.o + ((b * a.seq + t) * a.v_heads + hv) * a.v_dim + col, ot);
        r[i][j] = doc[row] == doc[kC - 1] ? r[i][j] * vec[kC + row] : 0.f;
      }
    const float all = vec[kC - 1];
    const bool cut = doc[kC - 1] != 0.f;
#pragma unroll
    for (int i = 0; i < KD / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = cut ? 0.f : S[i][j] * all;
    col_product<KD, NP>(keys + kPart, r, mixed, doc, doc[kC - 1], S);
    keys += 3 * kPart;
    tri += 2 * kTri * kPieces * kFrag;
    vec += 4 * kC;
  }
  if (a.h_last) store_state<KD>(a, a.h_last + bh * a.k_dim * a.v_dim, col, S);
}

template <typename T, int KD>
__global__ __launch_bounds__(64) void delta_bwd_kernel(Args<T> a) {
  constexpr int NP = kIn<T>, KS = KD / 32, kPart = KD / 8 * NP * kFrag;
  __shared__ float xs[kC][17];
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  const int tiles = a.v_pad / 16;
  const int64_t unit = xcd_order(blockIdx.x, gridDim.x), bh = unit / tiles;
  const int64_t b = bh / a.v_heads, hv = bh % a.v_heads, hk = hv / (a.v_heads / a.k_heads);
  const int col = (int)(unit % tiles) * 16 + m;
  const bool real = col < a.v_dim;
  floatx4 S[KD / 16];  // the gradient of the state after the chunk
  load_state<KD>(a, a.dh_last ? a.dh_last + bh * a.k_dim * a.v_dim : nullptr, col, S);
  for (int64_t c = a.chunks - 1; c >= 0; --c) {
    const uint16_t* keys = a.keys + ((b * a.k_heads + hk) * a.chunks + c) * (3 * kPart);
    const uint16_t* tri = a.tri + (bh * a.chunks + c) * (2 * kTri * kPieces * kFrag);
    const float* vec = a.vec + (bh * a.chunks + c) * (4 * kC);
    const float* doc = vec + 3 * kC;
    const bool mixed = doc[0] != doc[kC - 1], cut = doc[kC - 1] != 0.f;
    store_padded<KD>(a.dstates + (bh * a.chunks + c) * KD * a.v_pad + col, a.v_pad, S);
    floatx4 x[4], y[4], z[4];
    {
      bf16x8 sf[KS][kPieces];
#pragma unroll
      for (int s = 0; s < KS; ++s) split<kPieces>(S[2 * s], S[2 * s + 1], sf[s]);
      row_product<KS, NP>(keys, sf, y);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t t = c * kC + 16 * i + 4 * g + j;
        x[i][j] = real && t < a.seq
                      ? a.scale * load_scalar(a.d_o + ((b * a.seq + t) * a.v_heads + hv) * a.v_dim + col)
                      : 0.f;
      }
    tri_product<true>(tri + kTri * kPieces * kFrag, x, mixed, doc, xs, z);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 16 * i + 4 * g + j;
        if (doc[row] == doc[kC - 1]) z[i][j] = fmaf(vec[kC + row], y[i][j], z[i][j]);
      }
    tri_product<true>(tri, z, mixed, doc, xs, y);
    float* zs = a.z + (bh * a.chunks + c) * kC * a.v_pad + col;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 16 * i + 4 * g + j;
        const int64_t t = c * kC + row;
        zs[(int64_t)row * a.v_pad] = y[i][j];
        const float dv = vec[2 * kC + row] * y[i][j];
        if (real && t < a.seq)
          store_scalar(a.dv + ((b * a.seq + t) * a.v_heads + hv) * a.v_dim + col, dv);
        x[i][j] = doc[row] == 0.f ? x[i][j] * vec[row] : 0.f;
        y[i][j] = doc[row] == 0.f ? -dv * vec[row] : 0.f;
      }
    const float all = vec[kC - 1];
#pragma unroll
    for (int i = 0; i < KD / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = cut ? 0.f : S[i][j] * all;
    col_product<KD, NP>(keys + 2 * kPart, x, cut, doc, 0.f, S);
    col_product<KD, NP>(keys + kPart, y, cut, doc, 0.f, S);
  }
  if (a.dh0) store_state<KD>(a, a.dh0 + bh * a.k_dim * a.v_dim, col, S);
}

// ---------------------------------------------------------------------------
// The gradients of q, k, g and beta: a chunk of a value head to a workgroup of four waves, wave w the
// columns 16 w.. of everything turned (tokens as columns). Operands pass through LDS 32 columns of v_dim
// at a time, as fragments with their columns in order.
// ---------------------------------------------------------------------------
template <typename T, int KD>
struct GradShared {
  uint16_t u[4 * kPieces * kFrag], z[4 * kPieces * kFrag], d_o[4 * kIn<T> * kFrag];
  uint16_t S[KD / 16 * kPieces * kFrag], dS[KD / 16 * kPieces * kFrag];
  double G[kC];
  float beta[kC], dG[kC], w[kC], dbeta[kC], dot[4];
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
__global__ __launch_bounds__(256) void delta_grad_kernel(Args<T> a) {
  constexpr int NP = kIn<T>, MT = KD / 16, kPart = KD / 8 * NP * kFrag;
  __shared__ __attribute__((aligned(16))) GradShared<T, KD> s;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, m = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t unit = xcd_order(blockIdx.x, gridDim.x), chunk = unit % a.chunks, bh = unit / a.chunks;
  const int64_t b = bh / a.v_heads, hv = bh % a.v_heads, hk = hv / (a.v_heads / a.k_heads);
  const int64_t t0 = chunk * kC;
  if (w == 0) {
    const Gates x = chunk_gates(a, b, hv, t0);
    s.G[lane] = x.G;
    s.beta[lane] = x.beta;
    s.doc[lane] = x.doc;
  }
  __syncthreads();
  const int row = tid >> 2, c8 = tid & 3;  // what this thread stages
  const float* resid = a.resid + (unit * kC + row) * a.v_pad + 8 * c8;
  const float* zs = a.z + (unit * kC + row) * a.v_pad + 8 * c8;
  const float* st = a.states + (unit * KD + row) * a.v_pad + 8 * c8;
  const float* ds = a.dstates + (unit * KD + row) * a.v_pad + 8 * c8;
  const T* d_o = a.d_o + ((b * a.seq + t0 + row) * a.v_heads + hv) * a.v_dim;
  const bool in = t0 + row < a.seq;
  const float beta = s.beta[row];
  float dot_b = 0.f, dot_s = 0.f;

  // Slot n of the first w + 1: rows of u (tokens 16 n..) against the wave's columns of dO and of z; slot
  // n + 1 of the others: rows of dO and of z against its columns of u.
  floatx4 p[5] = {}, mm[5] = {}, dq[MT] = {}, ka[MT] = {}, kb[MT] = {};
  for (int v0 = 0; v0 < a.v_pad; v0 += 32) {
    __syncthreads();
    float x[8], y[8];
    load_vec<float, 8>(resid + v0, x);
    load_vec<float, 8>(zs + v0, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dot_b = fmaf(x[i], y[i], dot_b);
      x[i] *= beta;
    }
    stage<kPieces>(s.u, row, c8, x);
    stage<kPieces>(s.z, row, c8, y);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = v0 + 8 * c8 + 4 * h;
      float q[4] = {0.f, 0.f, 0.f, 0.f};
      if (in && at < a.v_dim) load_part(d_o, at, a.v_dim - at, q);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * h + i] = q[i];
    }
    stage<NP>(s.d_o, row, c8, x);
#pragma unroll
    for (int h = 0; h < (KD + 63) / 64; ++h)
      if (KD >= 64 || row < KD) {
        load_vec<float, 8>(st + (int64_t)64 * h * a.v_pad + v0, x);
        load_vec<float, 8>(ds + (int64_t)64 * h * a.v_pad + v0, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) dot_s = fmaf(x[i], y[i], dot_s);
        stage<kPieces>(s.S, row + 64 * h, c8, x);
        stage<kPieces>(s.dS, row + 64 * h, c8, y);
      }
    __syncthreads();
    bf16x8 uw[kPieces], zw[kPieces], ow[NP];
    load_frag(s.u + w * kPieces * kFrag, lane, uw);
    load_frag(s.z + w * kPieces * kFrag, lane, zw);
    load_frag(s.d_o + w * NP * kFrag, lane, ow);
#pragma unroll
    for (int n = 0; n < 5; ++n) {
      const bool turned = n <= w;
      if (turned) {
        bf16x8 un[kPieces];
        load_frag(s.u + n * kPieces * kFrag, lane, un);
        p[n] = mma(un, ow, p[n]);
        mm[n] = mma(un, zw, mm[n]);
      } else {
        bf16x8 zn[kPieces], on[NP];
        load_frag(s.d_o + (n - 1) * NP * kFrag, lane, on);
        load_frag(s.z + (n - 1) * kPieces * kFrag, lane, zn);
        p[n] = mma(on, uw, p[n]);
        mm[n] = mma(zn, uw, mm[n]);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      bf16x8 f[kPieces];
      load_frag(s.S + i * kPieces * kFrag, lane, f);
      dq[i] = mma(f, ow, dq[i]);
      ka[i] = mma(f, zw, ka[i]);
      load_frag(s.dS + i * kPieces * kFrag, lane, f);
      kb[i] = mma(f, uw, kb[i]);
    }
  }

  // The wave's column is token `mine`.
  const int mine = 16 * w + m, doc = s.doc[mine], last = s.doc[kC - 1];
  const double Gm = s.G[mine];
  const float bm = s.beta[mine];
  const float e = doc == 0 ? expf((float)Gm) : 0.f;
  const float et = doc == last ? expf((float)(s.G[kC - 1] - Gm)) : 0.f;
  const int64_t t = t0 + mine;
  const bool here = t < a.seq;
  const T* qrow = a.q + b * a.q_b + t * a.q_t + hk * a.q_h;
  const T* krow = a.k + b * a.k_b + t * a.k_t + hk * a.k_h;
  float wrote = 0.f;  // k . (dS' u)
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int d = 16 * i + 4 * g;
    float kv[4] = {0.f, 0.f, 0.f, 0.f};
    if (here && d < a.k_dim) load_part(krow, d, a.k_dim - d, kv);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      dq[i][r] = doc == 0 ? dq[i][r] * (a.scale * e) : 0.f;
      ka[i][r] = doc == 0 ? ka[i][r] * (-e * bm) : 0.f;
      kb[i][r] = doc == last ? kb[i][r] * et : 0.f;
      wrote = fmaf(kv[r], kb[i][r], wrote);
    }
  }
  // D dP (turned in the first w + 1 slots), and M.
#pragma unroll
  for (int n = 0; n < 5; ++n) {
    const bool turned = n <= w;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int other = 16 * (turned ? n : n - 1) + 4 * g + r;
      const bool one = s.doc[other] == doc && (turned ? other <= mine : other >= mine);
      const double G = s.G[other];
      const float D = one ? expf((float)(turned ? Gm - G : G - Gm)) : 0.f;
      const float bi = turned ? bm : s.beta[other];
      p[n][r] = one ? p[n][r] * (D * a.scale) : 0.f;
      mm[n][r] = one && other != mine ? mm[n][r] * (-bi * D) : 0.f;
    }
  }
  const uint16_t* kt = a.keys + ((b * a.k_heads + hk) * a.chunks + chunk) * (3 * kPart) + kPart;
  const uint16_t* qt = kt + kPart;
  const floatx4 none = {};
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    const int n = 2 * ks;
    if (n <= w) {  // turned: columns that this token reads
      bf16x8 pf[kPieces], mf[kPieces];
      split<kPieces>(p[n], n + 1 <= w ? p[n + 1] : none, pf);
      split<kPieces>(mm[n], n + 1 <= w ? mm[n + 1] : none, mf);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        bf16x8 f[NP];
        load_frag(kt + (i * 2 + ks) * NP * kFrag, lane, f);
        dq[i] = mma(f, pf, dq[i]);
        ka[i] = mma(f, mf, ka[i]);
      }
    }
    if (n + 1 >= w) {  // tokens that read this one
      bf16x8 pf[kPieces], mf[kPieces];
      split<kPieces>(n >= w ? p[n + 1] : none, p[n + 2], pf);
      split<kPieces>(n >= w ? mm[n + 1] : none, mm[n + 2], mf);
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
  float dG = 0.f;
  const bool shared = a.k_heads != a.v_heads;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int d = 16 * i + 4 * g;
    if (!here || d >= a.k_dim) continue;
    float qv[4], kv[4], dk[4], dqv[4];
    load_part(qrow, d, a.k_dim - d, qv);
    load_part(krow, d, a.k_dim - d, kv);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      dG = fmaf(qv[r], dq[i][r], dG);
      dG = fmaf(kv[r], ka[i][r] - kb[i][r], dG);
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
  dG += __shfl_xor(dG, 16);
  dG += __shfl_xor(dG, 32);
  wrote += __shfl_xor(wrote, 16);
  wrote += __shfl_xor(wrote, 32);
  if (g == 0) {
    s.dG[mine] = dG;
    s.w[mine] = wrote;
  }
  dot_b += lane_xor1(dot_b);
  dot_b += lane_xor2(dot_b);
  if (c8 == 0) s.dbeta[row] = dot_b;
  dot_s = wave_sum_all(dot_s);
  if (lane == 0) s.dot[w] = dot_s;
  __syncthreads();
  if (w == 0) {
    const int d = s.doc[lane];
    double v = s.dG[lane];
    float ends = wave_sum_all(s.w[lane]);  // zero for tokens of other documents than the last
    if (last == 0) ends = fmaf(expf((float)s.G[kC - 1]), (s.dot[0] + s.dot[1]) + (s.dot[2] + s.dot[3]), ends);
    if (lane == kC - 1) v += ends;
#pragma unroll
    for (int n = 1; n < 64; n *= 2) {
      const double after = __shfl_down(v, n);
      const int other = __shfl_down(d, n);
      if (lane + n < 64 && other == d) v += after;
    }
    const int before = __shfl_up(d, 1);
    if (d != (lane == 0 ? 0 : before)) v = 0.0;  // a document's first token: nothing decays into it
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
// l of wave w has columns 4 (l % 16).. of rows l / 16 + 4 w + 16 n.
// ---------------------------------------------------------------------------
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void delta_step_kernel(Args<T> a, float* h) {
  __shared__ float red[2][16][64];
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
  }
  // o = S_t^T q = p^T q + (q . k) beta r: both sums of the old state in one pass.
  float qk = 0.f;
  for (int d = tid & 63; d < a.k_dim; d += 64) qk = fmaf(load_scalar(q + d), load_scalar(k + d), qk);
  qk = wave_sum_all(qk);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    red[0][r0][c4 + c] = x[c];
    red[1][r0][c4 + c] = y[c];
  }
  __syncthreads();
  float wr[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    x[c] = y[c] = 0.f;
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      x[c] += red[0][n][c4 + c];
      y[c] += red[1][n][c4 + c];
    }
    const float v = c < left ? load_scalar(a.v + b * a.v_b + hv * a.v_h + col + c) : 0.f;
    wr[c] = beta * (v - x[c]);
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
