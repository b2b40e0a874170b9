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
// fp32. A value is two fp16 pieces, held to 2^-23 of itself or 2^-33, and a product three: off by 2e-6 at
// sides of 1024, 4.6e-6 at 12000 (a product of fp32 operands by 3e-6 and 7e-6). Matrices in bf16 may have one
// piece, where the caller leaves them that (from shorter sides of kOnePiece on: roundings average out over a
// side, and short ones take no less time with one): off by 1e-3 where bf16's own rounding is 1.7e-3, in 443 us
// for 744 to 805 (12 matrices of 1536 by 768), 1460 for 2290 to 2390 (the step of 8 blocks of width 512) or 1934
// for 4063 (8 of 2048 by 2048). X itself, which a X goes on from, keeps its second piece then too: weak
// directions grow 3.4 times a step by a X alone, and a rounding of X with them (a matrix of eight strong
// directions comes out off by 3e-4 of it, without that piece by 0.04, iterated in bf16 by 0.3; gradients with a
// sixteenth of strong directions by 8e-4).
#include <algorithm>
#include <atomic>
#include <climits>
#include <new>
#include <vector>

#include "mfma_tile.hpp"

namespace mqc {
namespace ortho {

using namespace mfma;

constexpr int kMatrices = 64, kGroups = 16;  // of a launch
constexpr float kScale = 256.f;              // (an fp16 number ends at 65504: values have to stay below 255)
constexpr int64_t kPartElems = 4096;         // elements that a workgroup adds the squares of
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
  int splits;            // workgroups that share a tile's columns in the first product
  int64_t shares;        // bytes: where their sums begin
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
  int side;     // of the first product's tiles
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

// The workgroup's group, the matrix in it and what is left of its number, `each` workgroups to a matrix;
// null for those that fill a group's last eight. An eighth of each group's go to an XCD, consecutive ones:
// tiles of one matrix share its rows in L2, and every XCD gets as much of the long shapes as of the short
// ones (in eighths of the whole launch, the longest of four shapes lay on one: 133 us for 80).
template <typename Each>
__device__ inline const Group* find(const Args& a, const Each& each, int& matrix, int& left) {
  const int at = blockIdx.x / kXCDs, xcd = blockIdx.x % kXCDs;
  int i = 0;
  while (i + 1 < a.count && at >= a.groups[i + 1].tiles) ++i;
  const Group& g = a.groups[i];
  const int n = each(g), rest = xcd * ((n * g.count + kXCDs - 1) / kXCDs) + at - g.tiles;
  matrix = rest / n;
  left = rest % n;
  return matrix < g.count && at - g.tiles < (n * g.count + kXCDs - 1) / kXCDs ? &g : nullptr;
}
template <typename T>
__device__ inline const T* source(const Args& a, const Group& g, int i) {
  return g.stack ? (const T*)a.matrices[g.first].g + i * g.stack : (const T*)a.matrices[g.first + i].g;
}
template <typename T>
__device__ inline T* target(const Args& a, const Group& g, int i) {
  return g.stack ? (T*)a.matrices[g.first].p + i * g.stack : (T*)a.matrices[g.first + i].p;
}

// --- momentum, and the sum of squares (42 M bf16 elements, fp32 momenta: 71 us, 5.9 TB/s) -----------------
template <bool MUON>
__device__ inline float update(const Args& a, float g, float m) {
  if constexpr (!MUON) return g;
  return a.nesterov ? fmaf(a.mu, m, (1.f - a.mu) * g) : m;
}

template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ortho_sum_kernel(Args a) {
  __shared__ double red[4];
  int i, part;
  const Group* group = find(a, [](const Group& g) { return g.sums; }, i, part);
  if (!group) return;
  const Group& g = *group;
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

// --- X_0 by rows and turned (of the same in pairs 151 us, 590 MB at 3.9 TB/s) ----------------------------
// Four values (times kScale) into a row, col a multiple of 4; the second pieces `second` bytes on (0: none).
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
  const Group* group =
      find(a, [](const Group& g) { return ceil_div(g.rows, 64) * ceil_div(g.cols, 64); }, i, left);
  if (!group) return;
  const Group& g = *group;
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
  const double scale = kScale / (total < a.eps ? (double)a.eps : total);  // (a norm may lie past fp32's ends)
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
    for (int k = 0; k < 4; ++k) v[k] = (float)(tile[r][q + k] * scale);
    if (r0 + r < g.rows) put4<PAIR>(straight + (r0 + r) * sp, c0 + q, v, tall ? second : none);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (float)(tile[q + k][r] * scale);
    if (c0 + r < g.cols) put4<PAIR>(turned + (c0 + r) * tp, r0 + q, v, tall ? none : second);
  }
}

// --- the products ------------------------------------------------------------------------------------------
// JOIN: the first product's tiles from the sums of those that shared their columns.
enum Stage { GRAM, JOIN, POLY, APPLY, LAST };

template <int S>
__host__ __device__ inline int symmetric_tiles(const Group& g) {
  const int t = ceil_div(g.m, S);
  return t * (t + 1) / 2;
}
template <int STAGE, int S>
__host__ __device__ inline int tile_count(const Group& g) {
  if (STAGE == GRAM) return symmetric_tiles<S>(g) * g.splits;
  if (STAGE == JOIN) return g.splits > 1 ? symmetric_tiles<64>(g) : 0;
  if (STAGE == POLY) return symmetric_tiles<S>(g);
  return ceil_div(g.m, S) * ceil_div(g.n, S);
}

// Stages in LDS. Launches of the smallest tiles have few of them on a CU to hide what a stage waits for (0.5 us
// of two stages, each of 16 KB): there three are under way.
constexpr int kSlots = 4;
template <typename Cfg>
constexpr int kLdsBytes = Cfg::TW == 64 ? kSlots * Cfg::kStageBytes : Cfg::kStagesBytes;

// Eight values of a row, col a multiple of 8; second pieces as in put4.
template <bool PAIR>
__device__ inline void put8(char* row, int col, const float (&v)[8], int64_t second = PAIR ? 64 : 0) {
  char* to = row + 2 * (PAIR ? col / 32 * 64 + col % 32 : col);
  u32x4 hi, lo;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    hi[c] = pack2<f16_t>(v[2 * c], v[2 * c + 1]);
    lo[c] = pack2<f16_t>(v[2 * c] - io<f16_t>::bits_to_f32(hi[c] & 0xffffu),
                         v[2 * c + 1] - io<f16_t>::bits_to_f32(hi[c] >> 16));
  }
  *(u32x4*)to = hi;
  if (second) *(u32x4*)(to + second) = lo;
}
// Eight values of a row, col a multiple of 8, and their sums.
template <bool PAIR>
__device__ inline void load8(const char* row, int col, u32x4 (&v)[2], int64_t second = PAIR ? 64 : 0) {
  const char* from = row + 2 * (PAIR ? col / 32 * 64 + col % 32 : col);
  v[0] = *(const u32x4*)from;
  v[1] = second ? *(const u32x4*)(from + second) : u32x4{0u, 0u, 0u, 0u};
}
__device__ inline float joined(const u32x4 (&v)[2], int c) {
  const uint32_t hi = v[0][c / 2], lo = v[1][c / 2];
  return io<f16_t>::bits_to_f32(c & 1 ? hi >> 16 : hi & 0xffffu) +
         io<f16_t>::bits_to_f32(c & 1 ? lo >> 16 : lo & 0xffffu);
}
// Eight elements of a matrix's row (its parameter's update where MUON).
template <typename T, bool MUON>
__device__ inline void put_result(T* to, int left, float (&v)[8], float decay, float rate) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (left <= 4 * h) break;
    float y[4], p[4];
    if constexpr (MUON) load_part((const T*)to, 4 * h, left - 4 * h, p);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      y[c] = v[4 * h + c] * (1.f / kScale);
      if constexpr (MUON) y[c] = fmaf(-rate, y[c], p[c] * decay);
    }
    store_part(to, 4 * h, left - 4 * h, y);
  }
}

// A tile's rows w of the left operand and x of the right one, S of each. What it leaves goes through LDS,
// the columns of a wave at a time: rows of x are written along w, and (the mirrored half of a symmetric
// product, X by rows, a wide matrix) rows of w along x, 16 bytes a lane. (Written from the registers, two
// bytes a lane, a step for the matrices of 8 blocks of width 512 took 2458 us in single pieces; with this,
// and long sides shared, 2034.) In pairs the symmetric products take 116 + 7 + 83 us of it a time, the last one
// 231: 60 GFLOP in three products, 0.78 PFLOP/s.
template <typename T, typename Cfg, bool PAIR, int STAGE, bool MUON>
__global__ __launch_bounds__(Cfg::kThreads, 2) void ortho_product_kernel(Args a) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  constexpr int S = Cfg::TW, XW = S / Cfg::NW_X, P = S + 4;
  static_assert(Cfg::TW == Cfg::TX && XW * P * 4 <= kLdsBytes<Cfg>, "square tiles, a wave's columns in LDS");
  constexpr bool SYMMETRIC = STAGE == GRAM || STAGE == JOIN || STAGE == POLY;
  int i, left;
  const Group* group = find(a, [](const Group& g) { return tile_count<STAGE, S>(g); }, i, left);
  if (!group) return;
  const Group& g = *group;
  char* ws = a.ws + g.base + i * g.each;
  int w0, x0, tile = 0, share = 0, k0 = 0;
  const char *W, *X;
  int wn = g.m, xn, K;
  if constexpr (SYMMETRIC) {
    if constexpr (STAGE == GRAM) share = left % g.splits, left /= g.splits;
    tile = left;
    int tw = (int)((sqrtf(8.f * (float)left + 1.f) - 1.f) * 0.5f);
    while (tw * (tw + 1) / 2 > left) --tw;
    while ((tw + 1) * (tw + 2) / 2 <= left) ++tw;
    w0 = tw * S, x0 = (left - tw * (tw + 1) / 2) * S;
    W = X = ws + (STAGE == POLY ? at_a<PAIR>(g, 0) : 0);
    xn = g.m, K = STAGE == POLY ? g.mp : g.np;
  } else {
    const int down = ceil_div(g.m, S);
    w0 = left % down * S, x0 = left / down * S;
    W = ws + at_a<PAIR>(g, 1), X = ws + at_xt<PAIR>(g, a.flip);
    xn = g.n, K = g.mp;
  }
  const int64_t rp = pitch<PAIR>(K);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  floatx4 acc[Cfg::WB][Cfg::XB];
#pragma unroll
  for (int u = 0; u < Cfg::WB; ++u)
#pragma unroll
    for (int v = 0; v < Cfg::XB; ++v) acc[u][v] = (floatx4){};
  // Where the lane's sums lie in the tile.
  const int wl = wave / Cfg::NW_X * (S / Cfg::NW_W) + 4 * (lane >> 4);
  const int xl = wave % Cfg::NW_X * XW + (lane & 15);
  // The sums of the workgroups that share a tile: [tile][share][x][w].
  if constexpr (STAGE == JOIN) {
    const int tw = w0 / a.side, tx = x0 / a.side, down = ceil_div(g.m, a.side);
    const int64_t each = (int64_t)a.side * a.side;
    const float* from = (const float*)(a.ws + g.shares) +
                        ((int64_t)i * (down * (down + 1) / 2) + tw * (tw + 1) / 2 + tx) * g.splits * each +
                        (int64_t)(x0 % a.side + xl) * a.side + w0 % a.side + wl;
    for (int s = 0; s < g.splits; ++s, from += each)
#pragma unroll
      for (int u = 0; u < Cfg::WB; ++u)
#pragma unroll
        for (int v = 0; v < Cfg::XB; ++v) acc[u][v] += *(const floatx4*)(from + 16 * v * a.side + 16 * u);
  } else {
    if constexpr (STAGE == GRAM) {
      const int steps = K / 64, each = ceil_div(steps, g.splits);
      k0 = share * each * 64;
      K = each * 64 < K - k0 ? each * 64 : K - k0;
    }
    // Rows past the matrix read its last one; what comes of them is not written.
    const auto rows = [&](const char* from, int r0, int count) {
      from += (int64_t)k0 * (PAIR ? 4 : 2);
      return [=](int gr, int k, int j, uint32_t& voff, const DmaLane& dl) -> const void* {
        const int base = r0 + gr < count ? r0 + gr : count - 1;
        const int r = r0 + gr + dl.lrow < count ? r0 + gr + dl.lrow : count - 1;
        voff = (uint32_t)((r - base) * rp) + dl.cb(j);
        return from + base * rp + (int64_t)k * 2;
      };
    };
    const int k2 = PAIR ? 2 * K : K;
    const auto wrow = rows(W, w0, wn), xrow = rows(X, x0, xn);
    if constexpr (S == 64) {
      const DmaLane dl(lane);
#pragma unroll
      for (int kt = 0; kt < kSlots - 1; ++kt) {
        if (kt * kBK >= k2) break;
        tile_issue_w<Cfg, kSlots>(kt, kt, wave, lds_addr(lds), dl, wrow);
        tile_issue_x<Cfg, kSlots>(kt, kt, wave, lds_addr(lds), dl, xrow);
      }
      tile_kloop_deep<Cfg, kSlots, kSlots, _Float16, PAIR>(k2, lds, acc, wrow, xrow);
    } else {
      tile_kloop_cfg<Cfg, _Float16, PAIR>(k2, lds, acc, wrow, xrow);
    }
  }
#pragma unroll
  for (int u = 0; u < Cfg::WB; ++u)
#pragma unroll
    for (int v = 0; v < Cfg::XB; ++v) acc[u][v] *= STAGE == JOIN ? 1.f : 1.f / kScale;
  if (STAGE == GRAM && g.splits > 1) {
    char* to = a.ws + g.shares +
               (((int64_t)i * symmetric_tiles<S>(g) + tile) * g.splits + share) * (S * S * 4);
    const uint32_t own = (uint32_t)(xl * S + wl) * 4;
#pragma unroll
    for (int v = 0; v < Cfg::XB; ++v, to += 16 * S * 4)
#pragma unroll
      for (int u = 0; u < Cfg::WB; ++u) *(floatx4*)(to + own + 64 * u) = acc[u][v];
    return;
  }

  // [x][w], the groups of eight columns in an order that both ways of reading find in distinct banks.
  float(*y)[P] = (float(*)[P])lds;
  const auto at8 = [](int x, int w) { return w ^ ((x >> 3 & 7) << 3); };
  constexpr int ITEMS = XW * (S / 8) / Cfg::kThreads;
  static_assert(XW * (S / 8) % Cfg::kThreads == 0, "whole items");
  const int64_t mpitch = pitch<PAIR>(g.mp), npitch = pitch<PAIR>(g.np), second = second_piece<PAIR>(g);
  const bool tall = g.rows > g.cols;
  char* xt = ws + at_xt<PAIR>(g, a.flip);
#pragma unroll 1
  for (int pass = 0; pass < Cfg::NW_X; ++pass) {
    const int xb = x0 + pass * XW;
    u32x4 old[ITEMS][2];
    if constexpr (STAGE == POLY || !SYMMETRIC) {
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        const int at = tid + it * Cfg::kThreads, x = xb + at / (S / 8), w = w0 + at % (S / 8) * 8;
        if (x >= xn || w >= g.mp) continue;
        if constexpr (STAGE == POLY) load8<PAIR>(ws + at_a<PAIR>(g, 0) + x * mpitch, w, old[it]);
        else load8<PAIR>(xt + x * mpitch, w, old[it], second);
      }
    }
    __syncthreads();  // the last stage, or the pass before, has been read
    if (wave % Cfg::NW_X == pass) {
#pragma unroll
      for (int u = 0; u < Cfg::WB; ++u)
#pragma unroll
        for (int v = 0; v < Cfg::XB; ++v) {
          const int x = 16 * v + (lane & 15);
          *(floatx4*)&y[x][at8(x, wl + 16 * u)] = acc[u][v];
        }
    }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int at = tid + it * Cfg::kThreads, xr = at / (S / 8), wr = at % (S / 8) * 8;
      const int x = xb + xr, w = w0 + wr;
      if (w >= g.mp) continue;
      float* from = &y[xr][at8(xr, wr)];
      float v[8];
      load_vec<float, 8>(from, v);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if constexpr (STAGE == POLY) v[c] = fmaf(a.c, v[c], a.b * joined(old[it], c));
        if constexpr (!SYMMETRIC) v[c] = fmaf(a.a, joined(old[it], c), v[c]);
        v[c] = w + c < wn && x < xn ? v[c] : 0.f;
      }
      if constexpr (STAGE == POLY || !SYMMETRIC) store_vec<float, 8>(from, v);
      if (x >= xn) continue;
      if constexpr (SYMMETRIC) put8<PAIR>(ws + at_a<PAIR>(g, STAGE == POLY) + x * mpitch, w, v);
      else if constexpr (STAGE == APPLY) put8<PAIR>(ws + at_xt<PAIR>(g, a.flip ^ 1) + x * mpitch, w, v, second);
      else if (tall && w < wn)
        put_result<T, MUON>(target<T>(a, g, i) + (int64_t)x * g.cols + w, wn - w, v, a.decay, g.rate);
    }
    if (SYMMETRIC ? w0 == x0 : STAGE == LAST && tall) continue;
    __syncthreads();
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int at = tid + it * Cfg::kThreads, wr = at / (XW / 8), xr = at % (XW / 8) * 8;
      const int x = xb + xr, w = w0 + wr;
      if (w >= wn || x >= (STAGE == LAST ? xn : SYMMETRIC ? g.mp : g.np)) continue;
      float v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = x + c < xn ? y[xr + c][at8(xr, wr)] : 0.f;
      if constexpr (SYMMETRIC) put8<PAIR>(ws + at_a<PAIR>(g, STAGE == POLY) + w * mpitch, x, v);
      else if constexpr (STAGE == APPLY) put8<PAIR>(ws + w * npitch, x, v);
      else put_result<T, MUON>(target<T>(a, g, i) + (int64_t)w * g.cols + x, xn - x, v, a.decay, g.rate);
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
using Tile64 = mfma::TileCfg<64, 64, 2, 2>;
using Tile128 = mfma::TileCfg<128, 128, 2, 2>;
using mfma::Tile256;

template <typename Count>
int64_t total(const Args& a, const Count& count) {
  int64_t n = 0;
  for (int i = 0; i < a.count; ++i) n += (int64_t)a.groups[i].count * count(a.groups[i]);
  return n;
}
// The side of a launch's tiles. The last product's are of 256 rows by 256 where they fill the card (half the
// bytes to LDS: with 8 matrices of 2048 x 2048 a call takes 4063 us in pairs for 4267 at 128, in single pieces
// 1934 for 2088; with two, of 128 such tiles, in single pieces 772 for 653), the symmetric ones, of fewer and
// with half a tile lost on the diagonal, of 128 (all at 256: 2136); where fewer than 128 of these are left, of 64.
template <int STAGE>
int tile_side(const Args& a) {
  if ((STAGE == ortho::APPLY || STAGE == ortho::LAST) && total(a, ortho::tile_count<STAGE, 256>) >= 256) return 256;
  return total(a, ortho::tile_count<STAGE, 128>) >= 128 ? 128 : 64;
}

// Where the groups' buffers and sums lie; returns the workspace's bytes. Long sides are shared among
// workgroups in the first product where its tiles alone would not fill the card (512 of 128 by 128), in
// shares of about as many columns as a workgroup has on average, at least 512; and of at most 8192, since an
// fp32 sum of n terms loses n^1/2: 70000 columns at once are off by 5.2e-6, in shares by less than 3.8e-6.
// (The products that sum over a shorter side are not shared: off by 4.2e-6 at 8400, 4.6e-6 at 12000, where
// products of fp32 operands are off by 6.5e-6 and 7.3e-6. Up to 2048 columns the launch that joins shares
// costs more than they save: 12 matrices of 768 by 1536 take 24 us in single pieces, shared 21 and 12.)
int64_t lay_out(Args& a, bool pair) {
  int64_t bytes = 0, parts = 0, steps = 0;
  for (int i = 0; i < a.count; ++i) {
    Group& g = a.groups[i];
    g.each = pair ? ortho::matrix_bytes<true>(g) : ortho::matrix_bytes<false>(g);
    g.base = bytes;
    bytes += g.each * g.count;
    g.parts = parts;
    parts += (int64_t)g.count * g.sums;
    g.splits = 1;
  }
  a.side = tile_side<ortho::POLY>(a);
  const int64_t slots = a.side == 128 ? 512 : 1024;
  const auto tiles = [&](const Group& g) -> int64_t {
    return a.side == 128 ? ortho::symmetric_tiles<128>(g) : ortho::symmetric_tiles<64>(g);
  };
  steps = total(a, [&](const Group& g) { return tiles(g) * (g.np / 64); });
  const int64_t least = std::max<int64_t>(8, (steps + slots - 1) / slots);
  for (int i = 0; i < a.count; ++i) {
    Group& g = a.groups[i];
    const int64_t have = g.np / 64;
    const int64_t want = have <= 32 ? 1 : std::max((have + least - 1) / least, (have + 127) / 128);
    const int64_t each = (have + want - 1) / want;
    g.splits = (int)((have + each - 1) / each);
    g.shares = bytes;
    if (g.splits > 1) bytes += g.count * tiles(g) * g.splits * a.side * a.side * 4;
  }
  a.sums = (double*)bytes;  // (an offset until the workspace is known)
  return bytes + (parts * 8 + 255) / 256 * 256;
}

// Workgroups of a launch, of which `each` are one matrix's: where each group's begin in an XCD. -1: too many.
template <typename Each>
int64_t number(Args& a, const Each& each, int64_t threads) {
  int64_t n = 0;
  for (int i = 0; i < a.count; ++i) {
    const int64_t of_group = (int64_t)a.groups[i].count * each(a.groups[i]);
    a.groups[i].tiles = (int)n;
    n += (of_group + kXCDs - 1) / kXCDs;
    if (of_group > INT_MAX - kXCDs || !launchable(n * kXCDs, threads)) return -1;
  }
  return n * kXCDs;
}

// Side of a stage's tiles (of the first product those that its shares were laid out for).
template <int STAGE>
int stage_side(const Args& a) {
  return STAGE == ortho::GRAM ? a.side : STAGE == ortho::JOIN ? 64 : tile_side<STAGE>(a);
}
template <int STAGE>
bool stage_fits(Args& a) {
  const int side = stage_side<STAGE>(a);
  return (side == 256   ? number(a, ortho::tile_count<STAGE, 256>, 512)
          : side == 128 ? number(a, ortho::tile_count<STAGE, 128>, 256)
                        : number(a, ortho::tile_count<STAGE, 64>, 256)) >= 0;
}
int64_t init_tiles(const Group& g) { return (int64_t)ortho::ceil_div(g.rows, 64) * ortho::ceil_div(g.cols, 64); }
// Whether all launches of a call can be made: known before the first, which changes momenta.
bool fits(Args a) {
  return number(a, [](const Group& g) { return g.sums; }, 256) >= 0 && number(a, init_tiles, 256) >= 0 &&
         stage_fits<ortho::GRAM>(a) && stage_fits<ortho::JOIN>(a) && stage_fits<ortho::POLY>(a) &&
         stage_fits<ortho::LAST>(a);
}

constexpr int kMaxDevices = 64;
template <typename T, typename Cfg, bool PAIR, int STAGE, bool MUON>
int launch_tiles(Args& a, hipStream_t s) {
  const int64_t n = number(a, ortho::tile_count<STAGE, Cfg::TW>, Cfg::kThreads);
  if (n < 0) return MQC_E_LIMIT;
  if (n == 0) return MQC_OK;
  const auto kernel = ortho::ortho_product_kernel<T, Cfg, PAIR, STAGE, MUON>;
  if (ortho::kLdsBytes<Cfg> > 65536) {  // has to be asked for, once on each device
    static std::atomic<bool> done[kMaxDevices];
    int device = -1;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return (int)e;
    if (device < 0 || device >= kMaxDevices) return MQC_E_LIMIT;
    if (!done[device]) {
      e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                              ortho::kLdsBytes<Cfg>);
      if (e != hipSuccess) return (int)e;
      done[device] = true;
    }
  }
  kernel<<<dim3((unsigned)n), dim3(Cfg::kThreads), ortho::kLdsBytes<Cfg>, s>>>(a);
  return launch_status();
}
template <typename T, bool PAIR, int STAGE, bool MUON>
int launch_product(Args& a, hipStream_t s) {
  const int side = stage_side<STAGE>(a);
  if constexpr (STAGE == ortho::APPLY || STAGE == ortho::LAST)
    if (side == 256) return launch_tiles<T, Tile256, PAIR, STAGE, MUON>(a, s);
  if constexpr (STAGE != ortho::JOIN)
    if (side == 128) return launch_tiles<T, Tile128, PAIR, STAGE, MUON>(a, s);
  return launch_tiles<T, Tile64, PAIR, STAGE, MUON>(a, s);
}

template <typename T, bool PAIR, bool MUON>
int iterate(Args& a, int steps, hipStream_t s) {
  int st = MQC_OK;
  a.flip = 0;
  for (int i = 0; i < steps && st == MQC_OK; ++i) {
    st = launch_product<float, PAIR, ortho::GRAM, false>(a, s);
    if (st == MQC_OK) st = launch_product<float, PAIR, ortho::JOIN, false>(a, s);
    if (st == MQC_OK) st = launch_product<float, PAIR, ortho::POLY, false>(a, s);
    if (st != MQC_OK) break;
    if (i + 1 < steps) {
      st = launch_product<float, PAIR, ortho::APPLY, false>(a, s);
      a.flip ^= 1;
    } else {
      st = launch_product<T, PAIR, ortho::LAST, MUON>(a, s);
    }
  }
  return st;
}

// A dtype of the C interface: the type, and whether bf16 matrices of any size are iterated in pairs.
int type_of(int64_t dtype) {
  const int64_t type = dtype & ~(int64_t)MQC_ORTHO_PAIRS;
  return type == MQC_F32 || type == MQC_BF16 || type == MQC_F16 ? (int)type : -1;
}
bool paired(int64_t dtype, int64_t rows, int64_t cols) {
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
  n = number(a, init_tiles, 256);
  if (n < 0) return MQC_E_LIMIT;
  ortho::ortho_init_kernel<T, PAIR, MUON><<<dim3((unsigned)n), dim3(256), 0, s>>>(a);
  st = launch_status();
  if (st != MQC_OK) return st;
  return iterate<T, PAIR, MUON>(a, steps, s);
}
template <bool MUON>
int run(Args& a, int dtype, int steps, char* ws, hipStream_t s) {
  const bool pair = paired(dtype, a.groups[0].rows, a.groups[0].cols);
  if (type_of(dtype) == MQC_F32) return run_pieces<float, true, MUON>(a, steps, ws, s);
  if (type_of(dtype) == MQC_F16) return run_pieces<f16_t, true, MUON>(a, steps, ws, s);
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
      if (type_of(rows[6 * i + 5]) == dtype && paired(rows[6 * i + 5], rows[6 * i + 3], rows[6 * i + 4]) == pair)
        order.push_back(i);
    std::stable_sort(order.begin(), order.end(), [&](int64_t x, int64_t y) {
      const int64_t *u = rows + 6 * x, *v = rows + 6 * y;
      const int64_t a = std::max(u[3], u[4]), b = std::max(v[3], v[4]);  // long ones begin first
      return a != b ? a > b : u[3] != v[3] ? u[3] < v[3] : u[4] < v[4];
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
      types.push_back(pair ? dtype | MQC_ORTHO_PAIRS : dtype);
    }
  }
}

int table(const int64_t* rows, int64_t count) {
  if (count < 0) return MQC_E_SHAPE;
  if (count > 0 && !rows) return MQC_E_NULL;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t* r = rows + 6 * i;
    if (type_of(r[5]) < 0) return MQC_E_DTYPE;
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
  if (type_of(dtype) < 0) return MQC_E_DTYPE;
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
  if (!fits(k)) return MQC_E_LIMIT;
  k.a = a, k.b = b, k.c = c, k.eps = eps;
  return run<false>(k, dtype, steps, (char*)workspace, (hipStream_t)stream);
}

extern "C" int64_t mqc_muon_workspace_bytes(const int64_t* matrices, int64_t count) {
  const int st = table(matrices, count);
  if (st != MQC_OK) return st;
  std::vector<Batch> work;
  std::vector<int> types;
  try {
    batches(matrices, count, 0.f, work, types);
  } catch (const std::bad_alloc&) {
    return MQC_E_LIMIT;
  }
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
  try {
    batches(matrices, count, rate, work, types);
  } catch (const std::bad_alloc&) {
    return MQC_E_LIMIT;
  }
  for (const Batch& w : work) {
    if (workspace_bytes < w.bytes) return MQC_E_SPACE;
    if (!fits(w.args)) return MQC_E_LIMIT;
  }
  const hipStream_t s = (hipStream_t)stream;
  for (size_t i = 0; i < work.size() && st == MQC_OK; ++i) {
    Args& k = work[i].args;
    k.a = a, k.b = b, k.c = c, k.eps = eps, k.mu = momentum, k.decay = decay, k.nesterov = nesterov;
    st = run<true>(k, types[i], steps, (char*)workspace, s);
  }
  return st;
}
