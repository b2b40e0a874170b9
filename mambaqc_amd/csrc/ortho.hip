// Orthogonalised updates of matrices: Newton's and Schulz's iteration, alone and as an optimiser's step
// with momentum.
//   m <- mu m + (1 - mu) g,  u = mu m + (1 - mu) g (or m),  X_0 = u / max(|u|_F, eps)
//   A = X X^T,  X <- a X + (b A + c A^2) X    (`steps` times)
//   p <- p decay - rate X
// An odd polynomial of X for its singular values, which it takes from below 1 to about 1; the iteration is
// on the shorter side m <= n (a tall matrix is turned as it is read and as it is written).
//
// All three products are of rows with their columns consecutive, tiles of mfma_tile.hpp's loop: A from
// rows of X, A^2 from rows of A, the last one from rows of B = b A + c A^2 and of X^T, so X is kept in both
// orders. A and B are symmetric: tiles below the diagonal are computed, those above it written as their
// mirrors. Every matrix of a call is in the same launches, whatever its shape.
//
// Operands are fp16 times 2^8 (X, A and B have values up to about 3, and most near n^-1/2), accumulators
// fp32. For matrices in fp32 and fp16 a value is two fp16 pieces, held to 2^-23 of itself or 2^-33, and a
// product three: off by 2e-6. For those in bf16 it is one (of shorter sides from kOnePiece on: roundings
// average out over a side, and short ones take no less time with one), but X itself, which a X goes on from, keeps its
// second piece: weak directions grow 3.4 times a step by a X alone, and a rounding of X with them (a matrix
// of eight strong directions comes out off by 3e-4 of it, without that piece by 0.04, iterated in bf16 by
// 0.3; gradients with a sixteenth of strong directions by 8e-4).
#include <algorithm>
#include <vector>

#include "mfma_tile.hpp"

namespace mqc {
namespace ortho {

using namespace mfma;

constexpr int kMatrices = 64, kGroups = 16;  // of a launch
constexpr float kScale = 256.f;
constexpr int64_t kPartElems = 16384;        // elements that a workgroup adds the squares of
constexpr int64_t kMaxParts = 256;
constexpr int kOnePiece = 256;

// Matrices of one shape.
struct Group {
  int64_t base, each;    // bytes: where the first one's buffers begin, and those of each
  int64_t stack;         // elements between matrices of a stack, 0: each has a row of the table
  int64_t parts;         // where its sums begin
  int rows, cols, m, n;  // m <= n, the sides
  int mp, np;            // padded to 64
  int count, first;      // matrices, and the first one's row
  int tiles;             // workgroups before this group's, by kernel
  int sums;              // workgroups that add a matrix's squares
  float rate;
};
struct Matrix {
  const void* g;
  void* p;
  float* m;
};
struct Args {
  Group groups[kGroups];
  Matrix matrices[kMatrices];
  int count;    // groups
  char* ws;
  double* sums;
  float a, b, c, eps, mu, decay;
  int nesterov;
  int flip;     // which X^T is read
};

template <bool PAIR>
__host__ __device__ inline int64_t pitch(int64_t k) { return k * (PAIR ? 4 : 2); }
// Buffers of a matrix: X by rows, X^T twice (and, where values are one piece, the second pieces of both,
// which no product reads), A, B.
template <bool PAIR>
__host__ __device__ inline int64_t at_xt(const Group& g, int which) {
  return g.m * pitch<PAIR>(g.np) + which * (int64_t)g.n * pitch<PAIR>(g.mp);
}
template <bool PAIR>
__host__ __device__ inline int64_t at_a(const Group& g, int which) {
  return at_xt<PAIR>(g, PAIR ? 2 : 4) + which * (int64_t)g.m * pitch<PAIR>(g.mp);
}
template <bool PAIR>
__host__ __device__ inline int64_t matrix_bytes(const Group& g) {
  return (at_a<PAIR>(g, 2) + 255) / 256 * 256;
}

// The workgroup's group, the matrix in it and what is left of its number, `each` workgroups to a matrix.
template <typename Each>
__device__ inline const Group& find(const Args& a, int64_t block, const Each& each, int& matrix, int& left) {
  int i = 0;
  while (i + 1 < a.count && block >= a.groups[i + 1].tiles) ++i;
  const Group& g = a.groups[i];
  const int n = each(g), rest = (int)block - g.tiles;
  matrix = rest / n;
  left = rest % n;
  return g;
}
template <typename T>
__device__ inline const T* source(const Args& a, const Group& g, int i) {
  return g.stack ? (const T*)a.matrices[g.first].g + i * g.stack : (const T*)a.matrices[g.first + i].g;
}
template <typename T>
__device__ inline T* target(const Args& a, const Group& g, int i) {
  return g.stack ? (T*)a.matrices[g.first].p + i * g.stack : (T*)a.matrices[g.first + i].p;
}

// --- momentum, and the sum of squares ------------------------------------------------------------------
template <bool MUON>
__device__ inline float update(const Args& a, float g, float m) {
  if constexpr (!MUON) return g;
  return a.nesterov ? fmaf(a.mu, m, (1.f - a.mu) * g) : m;
}

template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ortho_sum_kernel(Args a) {
  __shared__ double red[4];
  int i, part;
  const Group& g = find(a, blockIdx.x, [](const Group& g) { return g.sums; }, i, part);
  const int64_t n = (int64_t)g.rows * g.cols;
  const T* from = source<T>(a, g, i);
  float* mom = MUON ? a.matrices[g.first + i].m : nullptr;
  double sum = 0.0;
  const int64_t step = (int64_t)g.sums * 1024;
  for (int64_t at = (int64_t)part * 1024 + threadIdx.x * 4; at < n; at += step) {
    const int left = (int)(n - at < 4 ? n - at : 4);
    float v[4] = {}, m[4] = {};
    load_part(from + at, 0, left, v);
    if constexpr (MUON) {
      load_part((const float*)mom + at, 0, left, m);
#pragma unroll
      for (int c = 0; c < 4; ++c) m[c] = fmaf(a.mu, m[c], (1.f - a.mu) * v[c]);
      store_part(mom + at, 0, left, m);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const double u = update<MUON>(a, v[c], m[c]);
      if (c < left) sum = fma(u, u, sum);
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.sums[g.parts + (int64_t)i * g.sums + part] = (red[0] + red[1]) + (red[2] + red[3]);
}

// --- X_0 by rows and turned ------------------------------------------------------------------------------
// One value (times kScale) into a row.
template <bool PAIR>
__device__ inline void put(char* row, int col, float v) {
  _Float16* to = (_Float16*)row + (PAIR ? col / 32 * 64 + col % 32 : col);
  const _Float16 hi = (_Float16)v;
  to[0] = hi;
  if constexpr (PAIR) to[32] = (_Float16)(v - (float)hi);
}
// Four of them, col a multiple of 4; the second pieces `second` bytes on (0: none).
__device__ inline float half_of(const u32x2& v, int c) {
  return io<f16_t>::bits_to_f32(c & 1 ? v[c / 2] >> 16 : v[c / 2] & 0xffffu);
}
template <bool PAIR>
__device__ inline void put4(char* row, int col, const float (&v)[4], int64_t second = PAIR ? 64 : 0) {
  char* to = row + 2 * (PAIR ? col / 32 * 64 + col % 32 : col);
  const u32x2 hi = {pack2<f16_t>(v[0], v[1]), pack2<f16_t>(v[2], v[3])};
  *(u32x2*)to = hi;
  if (second) {
    float r[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) r[c] = v[c] - half_of(hi, c);
    *(u32x2*)(to + second) = u32x2{pack2<f16_t>(r[0], r[1]), pack2<f16_t>(r[2], r[3])};
  }
}
template <bool PAIR>
__device__ inline void get4(const char* row, int col, float (&v)[4], int64_t second = PAIR ? 64 : 0) {
  const char* from = row + 2 * (PAIR ? col / 32 * 64 + col % 32 : col);
  const u32x2 hi = *(const u32x2*)from;
  u32x2 lo = {0u, 0u};
  if (second) lo = *(const u32x2*)(from + second);
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = half_of(hi, c) + half_of(lo, c);
}
// From a value of X^T to its second piece.
template <bool PAIR>
__device__ inline int64_t second_piece(const Group& g) {
  return PAIR ? 64 : 2 * (int64_t)g.n * pitch<PAIR>(g.mp);
}

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <typename T, bool PAIR, bool MUON>
__global__ __launch_bounds__(256) void ortho_init_kernel(Args a) {
  __shared__ float tile[64][65];
  __shared__ double total;
  int i, left;
  const Group& g = find(a, blockIdx.x,
                        [](const Group& g) { return ceil_div(g.rows, 64) * ceil_div(g.cols, 64); }, i, left);
  if (threadIdx.x < 64) {
    double s = 0.0;
    for (int k = threadIdx.x; k < g.sums; k += 64) s += a.sums[g.parts + (int64_t)i * g.sums + k];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
    if (threadIdx.x == 0) total = sqrt(s);
  }
  const int across = ceil_div(g.cols, 64), r0 = left / across * 64, c0 = left % across * 64;
  const T* from = source<T>(a, g, i);
  const float* mom = MUON ? a.matrices[g.first + i].m : nullptr;
  const int c = threadIdx.x & 63;
  for (int r = threadIdx.x >> 6; r < 64; r += 4) {
    float v = 0.f;
    if (r0 + r < g.rows && c0 + c < g.cols) {
      const int64_t at = (int64_t)(r0 + r) * g.cols + c0 + c;
      v = update<MUON>(a, load_scalar(from + at), MUON ? mom[at] : 0.f);
    }
    tile[r][c] = v;
  }
  __syncthreads();
  const float norm = (float)total, scale = kScale / (norm < a.eps ? a.eps : norm);
  char* ws = a.ws + g.base + i * g.each;
  const bool tall = g.rows > g.cols;
  // By the rows of what was read, and turned.
  char* straight = ws + (tall ? at_xt<PAIR>(g, 0) : 0);
  char* turned = ws + (tall ? 0 : at_xt<PAIR>(g, 0));
  const int64_t sp = pitch<PAIR>(tall ? g.mp : g.np), tp = pitch<PAIR>(tall ? g.np : g.mp);
  const int q = (threadIdx.x & 15) * 4;
  const int64_t second = second_piece<PAIR>(g), none = PAIR ? 64 : 0;
  for (int r = threadIdx.x >> 4; r < 64; r += 16) {
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = tile[r][q + k] * scale;
    if (r0 + r < g.rows) put4<PAIR>(straight + (r0 + r) * sp, c0 + q, v, tall ? second : none);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = tile[q + k][r] * scale;
    if (c0 + r < g.cols) put4<PAIR>(turned + (c0 + r) * tp, r0 + q, v, tall ? none : second);
  }
}

// --- the products ------------------------------------------------------------------------------------------
enum Stage { GRAM, POLY, APPLY, LAST };

template <int STAGE, int T>
__host__ __device__ inline int tile_count(const Group& g) {
  const int t = ceil_div(g.m, T);
  return STAGE == GRAM || STAGE == POLY ? t * (t + 1) / 2 : t * ceil_div(g.n, T);
}

template <typename T, typename Cfg, bool PAIR, int STAGE, bool MUON>
__global__ __launch_bounds__(Cfg::kThreads) void ortho_product_kernel(Args a) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  constexpr int S = Cfg::TW;
  static_assert(Cfg::TW == Cfg::TX, "square tiles");
  const int64_t n = gridDim.x, lin = blockIdx.x;
  const int64_t block = n % kXCDs ? lin : (lin % kXCDs) * (n / kXCDs) + lin / kXCDs;
  int i, left;
  const Group& g = find(a, block, [](const Group& g) { return tile_count<STAGE, S>(g); }, i, left);
  char* ws = a.ws + g.base + i * g.each;
  // Rows of both operands (w: four consecutive ones to a lane).
  int w0, x0;
  const char *W, *X;
  int wn, xn, K;
  bool turned = false;
  if constexpr (STAGE == GRAM || STAGE == POLY) {
    int tw = (int)((sqrtf(8.f * (float)left + 1.f) - 1.f) * 0.5f);
    while (tw * (tw + 1) / 2 > left) --tw;
    while ((tw + 1) * (tw + 2) / 2 <= left) ++tw;
    w0 = tw * S, x0 = (left - tw * (tw + 1) / 2) * S;
    W = X = ws + (STAGE == GRAM ? 0 : at_a<PAIR>(g, 0));
    wn = xn = g.m, K = STAGE == GRAM ? g.np : g.mp;
  } else {
    const int down = ceil_div(g.m, S), tm = left % down, tn = left / down;
    W = ws + at_a<PAIR>(g, 1), X = ws + at_xt<PAIR>(g, a.flip);
    w0 = tm * S, x0 = tn * S, wn = g.m, xn = g.n, K = g.mp;
    // The last product's lanes write along the rows of the matrix: of a wide one X^T's rows come first.
    turned = STAGE == LAST && g.rows <= g.cols;
    if (turned) {
      const char* o = W;
      W = X, X = o;
      w0 = tn * S, x0 = tm * S, wn = g.n, xn = g.m;
    }
  }
  const int64_t rp = pitch<PAIR>(K);
  floatx4 acc[Cfg::WB][Cfg::XB];
#pragma unroll
  for (int u = 0; u < Cfg::WB; ++u)
#pragma unroll
    for (int v = 0; v < Cfg::XB; ++v) acc[u][v] = (floatx4){};
  // Rows past the matrix read its last one; what comes of them is not written.
  const auto rows = [&](const char* from, int r0, int count) {
    return [=](int gr, int k0, int j, uint32_t& voff, const DmaLane& dl) -> const void* {
      const int base = r0 + gr < count ? r0 + gr : count - 1;
      const int r = r0 + gr + dl.lrow < count ? r0 + gr + dl.lrow : count - 1;
      voff = (uint32_t)((r - base) * rp) + dl.cb(j);
      return from + base * rp + (int64_t)k0 * 2;
    };
  };
  tile_kloop_cfg<Cfg, _Float16, PAIR>(PAIR ? 2 * K : K, lds, acc, rows(W, w0, wn), rows(X, x0, xn));

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = w0 + wave / Cfg::NW_X * (S / Cfg::NW_W) + 4 * (lane >> 4);
  const int xr = x0 + wave % Cfg::NW_X * (S / Cfg::NW_X) + (lane & 15);
  const int64_t mpitch = pitch<PAIR>(g.mp);
#pragma unroll
  for (int u = 0; u < Cfg::WB; ++u)
#pragma unroll
    for (int v = 0; v < Cfg::XB; ++v) {
      const int w = wr + 16 * u, x = xr + 16 * v;
      if (x >= xn) continue;
      float y[4], old[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) y[c] = acc[u][v][c] * (1.f / kScale);
      if constexpr (STAGE == GRAM || STAGE == POLY) {
        if (w >= g.mp) continue;
        char* to = ws + at_a<PAIR>(g, STAGE == POLY);
        if constexpr (STAGE == POLY) get4<PAIR>(ws + at_a<PAIR>(g, 0) + x * mpitch, w, old);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if constexpr (STAGE == POLY) y[c] = fmaf(a.c, y[c], a.b * old[c]);
          if (w + c >= wn) y[c] = 0.f;
        }
        put4<PAIR>(to + x * mpitch, w, y);
        if (w0 != x0) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (w + c < wn) put<PAIR>(to + (w + c) * mpitch, x, y[c]);
        }
      } else if constexpr (STAGE == APPLY) {
        if (w >= g.mp) continue;
        get4<PAIR>(ws + at_xt<PAIR>(g, a.flip) + x * mpitch, w, old, second_piece<PAIR>(g));
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = w + c < wn ? fmaf(a.a, old[c], y[c]) : 0.f;
        put4<PAIR>(ws + at_xt<PAIR>(g, a.flip ^ 1) + x * mpitch, w, y, second_piece<PAIR>(g));
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (w + c < wn) put<PAIR>(ws + (w + c) * pitch<PAIR>(g.np), x, y[c]);
      } else {
        if (w >= wn) continue;
        const char* from = ws + at_xt<PAIR>(g, a.flip);
        if (turned) {
          const char* at = from + 2 * (PAIR ? x / 32 * 64 + x % 32 : x);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const _Float16* one = (const _Float16*)(at + (w + c < wn ? w + c : w) * mpitch);
            old[c] = (float)one[0] + (float)one[second_piece<PAIR>(g) / 2];
          }
        } else {
          get4<PAIR>(from + x * mpitch, w, old, second_piece<PAIR>(g));
        }
        T* to = target<T>(a, g, i) + (int64_t)x * g.cols;
        const int most = wn - w;
        float p[4];
        if constexpr (MUON) load_part((const T*)to, w, most, p);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          y[c] = fmaf(a.a, old[c], y[c]) * (1.f / kScale);
          if constexpr (MUON) y[c] = fmaf(-g.rate, y[c], p[c] * a.decay);
        }
        store_part(to, w, most, y);
      }
    }
}

}  // namespace ortho
}  // namespace mqc

using namespace mqc;

namespace {

using ortho::Args;
using ortho::Group;

// How the tables of a call become launches: matrices of one type, at most kMatrices of kGroups shapes.
struct Batch {
  Args args;
  int64_t bytes;  // of workspace
};
constexpr int64_t kMaxSide = 32768, kMaxLong = 1 << 24;

int shape(int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1) return MQC_E_SHAPE;
  if (std::min(rows, cols) > kMaxSide || std::max(rows, cols) > kMaxLong) return MQC_E_LIMIT;
  return MQC_OK;
}
Group group_of(int64_t rows, int64_t cols) {
  Group g{};
  g.rows = (int)rows, g.cols = (int)cols;
  g.m = (int)std::min(rows, cols), g.n = (int)std::max(rows, cols);
  g.mp = (g.m + 63) / 64 * 64, g.np = (g.n + 63) / 64 * 64;
  const int64_t parts = (rows * cols + ortho::kPartElems - 1) / ortho::kPartElems;
  g.sums = (int)std::min(parts, ortho::kMaxParts);
  return g;
}
// Where the groups' buffers and sums lie; returns the workspace's bytes.
int64_t lay_out(Args& a, bool pair) {
  int64_t bytes = 0, parts = 0;
  for (int i = 0; i < a.count; ++i) {
    Group& g = a.groups[i];
    g.each = pair ? ortho::matrix_bytes<true>(g) : ortho::matrix_bytes<false>(g);
    g.base = bytes;
    bytes += g.each * g.count;
    g.parts = parts;
    parts += (int64_t)g.count * g.sums;
  }
  a.sums = (double*)bytes;  // (an offset until the workspace is known)
  return bytes + (parts * 8 + 255) / 256 * 256;
}

// Workgroups of a launch, of which `each` are one matrix's: where each group's begin. -1: too many.
template <typename Each>
int64_t number(Args& a, const Each& each, int64_t threads) {
  int64_t n = 0;
  for (int i = 0; i < a.count; ++i) {
    a.groups[i].tiles = (int)n;
    n += (int64_t)a.groups[i].count * each(a.groups[i]);
    if (!launchable(n, threads)) return -1;
  }
  return n;
}

template <typename T, typename Cfg, bool PAIR, int STAGE, bool MUON>
int launch_product(Args& a, hipStream_t s) {
  const int64_t n = number(a, ortho::tile_count<STAGE, Cfg::TW>, Cfg::kThreads);
  if (n < 0) return MQC_E_LIMIT;
  ortho::ortho_product_kernel<T, Cfg, PAIR, STAGE, MUON>
      <<<dim3((unsigned)n), dim3(Cfg::kThreads), Cfg::kStagesBytes, s>>>(a);
  return launch_status();
}

template <typename T, typename Cfg, bool PAIR, bool MUON>
int iterate(Args& a, int steps, hipStream_t s) {
  int st = MQC_OK;
  a.flip = 0;
  for (int i = 0; i < steps && st == MQC_OK; ++i) {
    st = launch_product<float, Cfg, PAIR, ortho::GRAM, false>(a, s);
    if (st == MQC_OK) st = launch_product<float, Cfg, PAIR, ortho::POLY, false>(a, s);
    if (st != MQC_OK) break;
    if (i + 1 < steps) {
      st = launch_product<float, Cfg, PAIR, ortho::APPLY, false>(a, s);
      a.flip ^= 1;
    } else {
      st = launch_product<T, Cfg, PAIR, ortho::LAST, MUON>(a, s);
    }
  }
  return st;
}

using Small = mfma::TileCfg<64, 64, 2, 2>;
using Large = mfma::TileCfg<128, 128, 2, 2>;

bool paired(int dtype, int64_t rows, int64_t cols) {
  return dtype != MQC_BF16 || std::min(rows, cols) < ortho::kOnePiece;
}

template <typename T, bool PAIR, bool MUON>
int run_pieces(Args& a, int steps, char* ws, hipStream_t s) {
  a.ws = ws;
  a.sums = (double*)(ws + (int64_t)a.sums);
  int64_t n = number(a, [](const Group& g) { return g.sums; }, 256);
  if (n < 0) return MQC_E_LIMIT;
  ortho::ortho_sum_kernel<T, MUON><<<dim3((unsigned)n), dim3(256), 0, s>>>(a);
  int st = launch_status();
  if (st != MQC_OK) return st;
  n = number(a, [](const Group& g) { return ortho::ceil_div(g.rows, 64) * ortho::ceil_div(g.cols, 64); }, 256);
  if (n < 0) return MQC_E_LIMIT;
  ortho::ortho_init_kernel<T, PAIR, MUON><<<dim3((unsigned)n), dim3(256), 0, s>>>(a);
  st = launch_status();
  if (st != MQC_OK) return st;
  const int64_t large = number(a, ortho::tile_count<ortho::GRAM, Large::TW>, Large::kThreads);
  return large >= 128 ? iterate<T, Large, PAIR, MUON>(a, steps, s) : iterate<T, Small, PAIR, MUON>(a, steps, s);
}
template <bool MUON>
int run(Args& a, int dtype, int steps, char* ws, hipStream_t s) {
  const bool pair = paired(dtype, a.groups[0].rows, a.groups[0].cols);
  if (dtype == MQC_F32) return run_pieces<float, true, MUON>(a, steps, ws, s);
  if (dtype == MQC_F16) return run_pieces<f16_t, true, MUON>(a, steps, ws, s);
  return pair ? run_pieces<bf16_t, true, MUON>(a, steps, ws, s) : run_pieces<bf16_t, false, MUON>(a, steps, ws, s);
}

int factors(int steps, float eps) { return steps < 1 || steps > 100 || !(eps >= 0.f) ? MQC_E_SHAPE : MQC_OK; }

// A table of matrices (rows of six values: p, grad, m, rows, cols, dtype) in launches: by type and pieces,
// and in these by shape. The workspace is that of the largest.
void batches(const int64_t* rows, int64_t count, float rate, std::vector<Batch>& out,
            std::vector<int>& types) {
  for (int kind = 0; kind < 4; ++kind) {
    const int dtype = kind == 0 ? MQC_F32 : kind == 1 ? MQC_F16 : MQC_BF16;
    const bool pair = kind < 3;
    std::vector<int64_t> order;
    for (int64_t i = 0; i < count; ++i)
      if (rows[6 * i + 5] == dtype && paired(dtype, rows[6 * i + 3], rows[6 * i + 4]) == pair)
        order.push_back(i);
    std::stable_sort(order.begin(), order.end(), [&](int64_t x, int64_t y) {
      const int64_t *u = rows + 6 * x, *v = rows + 6 * y;
      return u[3] != v[3] ? u[3] < v[3] : u[4] < v[4];
    });
    size_t at = 0;
    while (at < order.size()) {
      Batch b{};
      int used = 0;
      for (; at < order.size() && used < ortho::kMatrices; ++at) {
        const int64_t* r = rows + 6 * order[at];
        Group* g = b.args.count ? &b.args.groups[b.args.count - 1] : nullptr;
        if (!g || g->rows != r[3] || g->cols != r[4]) {
          if (b.args.count == ortho::kGroups) break;
          g = &b.args.groups[b.args.count++];
          *g = group_of(r[3], r[4]);
          g->first = used;
          g->rate = rate * (r[3] > r[4] ? std::sqrt((float)r[3] / (float)r[4]) : 1.f);
        }
        ++g->count;
        b.args.matrices[used++] = {(const void*)r[1], (void*)r[0], (float*)r[2]};
      }
      b.bytes = lay_out(b.args, pair);
      out.push_back(b);
      types.push_back(dtype);
    }
  }
}

int table(const int64_t* rows, int64_t count) {
  if (count < 0) return MQC_E_SHAPE;
  if (count > 0 && !rows) return MQC_E_NULL;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t* r = rows + 6 * i;
    if (r[5] != MQC_F32 && r[5] != MQC_BF16 && r[5] != MQC_F16) return MQC_E_DTYPE;
    const int st = shape(r[3], r[4]);
    if (st != MQC_OK) return st;
  }
  return MQC_OK;
}

Args one_stack(const void* x, void* out, int64_t batch, int64_t rows, int64_t cols) {
  Args a{};
  a.count = 1;
  a.groups[0] = group_of(rows, cols);
  a.groups[0].count = (int)batch;
  a.groups[0].stack = rows * cols;
  a.matrices[0] = {x, out, nullptr};
  return a;
}

}  // namespace

extern "C" int64_t mqc_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int dtype) {
  if (batch < 0) return MQC_E_SHAPE;
  const int st = shape(rows, cols);
  if (st != MQC_OK) return st;
  if (dtype != MQC_F32 && dtype != MQC_BF16 && dtype != MQC_F16) return MQC_E_DTYPE;
  if (batch > 65535) return MQC_E_LIMIT;
  Args a = one_stack(nullptr, nullptr, batch, rows, cols);
  return lay_out(a, paired(dtype, rows, cols));
}

extern "C" int mqc_orthogonalize(const void* x, void* out, int64_t batch, int64_t rows, int64_t cols,
                                 int steps, float a, float b, float c, float eps, int dtype,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t bytes = mqc_orthogonalize_workspace_bytes(batch, rows, cols, dtype);
  if (bytes < 0) return (int)bytes;
  const int st = factors(steps, eps);
  if (st != MQC_OK) return st;
  if (batch == 0) return MQC_OK;
  if (!x || !out || !workspace) return MQC_E_NULL;
  if (workspace_bytes < bytes) return MQC_E_SPACE;
  if (!aligned(workspace, 256)) return MQC_E_ALIGN;
  Args k = one_stack(x, out, batch, rows, cols);
  lay_out(k, paired(dtype, rows, cols));
  k.a = a, k.b = b, k.c = c, k.eps = eps;
  return run<false>(k, dtype, steps, (char*)workspace, (hipStream_t)stream);
}

extern "C" int64_t mqc_muon_workspace_bytes(const int64_t* matrices, int64_t count) {
  const int st = table(matrices, count);
  if (st != MQC_OK) return st;
  std::vector<Batch> work;
  std::vector<int> types;
  batches(matrices, count, 0.f, work, types);
  int64_t most = 0;
  for (const Batch& b : work) most = std::max(most, b.bytes);
  return most;
}

extern "C" int mqc_muon_step(const int64_t* matrices, int64_t count, float decay, float rate,
                             float momentum, int nesterov, int steps, float a, float b, float c, float eps,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  int st = table(matrices, count);
  if (st == MQC_OK) st = factors(steps, eps);
  if (st != MQC_OK) return st;
  if (count == 0) return MQC_OK;
  for (int64_t i = 0; i < count; ++i)
    if (!matrices[6 * i] || !matrices[6 * i + 1] || !matrices[6 * i + 2]) return MQC_E_NULL;
  if (!workspace) return MQC_E_NULL;
  if (!aligned(workspace, 256)) return MQC_E_ALIGN;
  std::vector<Batch> work;
  std::vector<int> types;
  batches(matrices, count, rate, work, types);
  for (const Batch& w : work)
    if (workspace_bytes < w.bytes) return MQC_E_SPACE;
  const hipStream_t s = (hipStream_t)stream;
  for (size_t i = 0; i < work.size() && st == MQC_OK; ++i) {
    Args& k = work[i].args;
    k.a = a, k.b = b, k.c = c, k.eps = eps, k.mu = momentum, k.decay = decay, k.nesterov = nesterov;
    st = run<true>(k, types[i], steps, (char*)workspace, s);
  }
  return st;
}
