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

// The exponents are held in base 2: p_t = log2(e) D_t exp(log_rate), a_t = 2^-p_t.
//
// Time is cut into chunks, a chunk into one span of steps for each of its waves, and a lane walks one
// channel of its wave's span: first from zero (u, its last state, and the sum of p, which give what the
// span makes of any state before it), then, once the state before the span is known, through the
// states themselves: inputs are read once, and their gates computed once. The spans of a chunk join in
// LDS. Between chunks the state goes through memory within the launch: see scan_entry.
//
// What bounds it: 8 bytes an element forward and 14 backward (bf16) against some 33 and 58 vector
// instructions (5 and 6 of which take four times as long), so neither memory (a copy's 5.1 TB/s) nor
// arithmetic alone, but how well workgroups overlap. The kernels alone, bf16: a prompt of 16384 x 1536 48 us
// (201 MB, 4.2 TB/s; loads and stores alone 32, with LDS and the words between chunks 38); 4 x 2048 x 1536
// forward 25 us, backward 41 (176 MB, 4.3 TB/s); past the last cache, 1 x 65536 x 1536 203 and 381. fp32: 81
// (403 MB, 5.0 TB/s), 33 and 57 (352 MB, 6.2 TB/s).
// Spans and waves, same prompt: 8 of 16 steps 47, 8 of 8 66, 4 of 16 68, 4 of 32 52, 16 of 8 62; backward
// of 4 x 2048 x 1536 (before later stages): 8 waves of 8 steps 53, 4 of 16 45, 4 of 32 65. Chunks joined one
// by one: 8 or 16 47, 32 49, 64 55. Not kept: workgroups that stay and load the next chunk ahead (61 to
// 82: they all wait for one another in turn), spans walked for a guessed chunk while the counter answers
// (56 to 77: it guesses wrong), 64 registers a lane for four workgroups a CU (51 to 57).
constexpr int kScanLanes = 64;  // channels of a workgroup
constexpr int kScanWaves = 8;   // spans of a chunk, forward
constexpr int kScanSteps = 16;  // steps of a span
constexpr int kBackWaves = 4;   // and backward (whose steps take three times the registers)
constexpr int kBackSteps = 16;
constexpr int kScanChunk = kBackWaves * kBackSteps;  // steps between the states that training stores
constexpr int kScanGroup = 16;  // chunks that are joined one by one (scan_entry)
static_assert(kScanWaves * kScanSteps % kScanChunk == 0 && kScanChunk % kScanSteps == 0, "stored states");

// log2(1 + 2^v): what rounding 1 + e leaves of e is added to first order.
__device__ inline float scan_softplus2(float v, float& e, float& u) {
  e = __builtin_amdgcn_exp2f(-fabsf(v));
  u = 1.f + e;
  return fmaf(e - (u - 1.f), 1.44269504f, fmaxf(v, 0.f) + __builtin_amdgcn_logf(u));
}

// 1 - 2^-p for p up to 1, by a minimax fit of (1 - 2^-p) / p (off by 2^-26.6, rounded by 2^-23).
__device__ inline float scan_slow(float p) {
  float w = fmaf(p, -1.14580565e-4f, 1.29078003e-3f);
  w = fmaf(p, w, -9.5962761e-3f);
  w = fmaf(p, w, 5.5498954e-2f);
  w = fmaf(p, w, -2.40226060e-1f);
  w = fmaf(p, w, 6.93147182e-1f);
  return p * w;
}
// A step's a and w = 1 - a, each to a few 2^-24 of itself.
__device__ inline void scan_pair(float p, float& a, float& w) {
  a = __builtin_amdgcn_exp2f(-p);
  const float slow = scan_slow(p);  // (in every lane: a branch here keeps steps from overlapping)
  w = p < 1.f ? slow : 1.f - a;
}
// A slow channel has a near 1 and forgets by 1 - a a token: an a rounded to fp32 shifts its rate, and
// with it the gain at rest, by up to 2^-24 / (1 - a). A span's walk takes a as it is, which adds up over
// 16 steps (2^-20); the decay of a span and of more is kept as one number, c = 1 - a where a is over a
// half and -a otherwise; the sign bit tells.
__device__ inline bool scan_fast(float c) { return __float_as_int(c) < 0; }  // c is -a
__device__ inline float scan_a(float c) { return scan_fast(c) ? -c : 1.f - c; }
__device__ inline float scan_w(float c) { return scan_fast(c) ? 1.f + c : c; }
// a v.
__device__ inline float scan_fade(float c, float v) { return fmaf(-c, v, scan_fast(c) ? 0.f : v); }
__device__ inline bool scan_finite(float v) { return fabsf(v) < __builtin_inff(); }

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
struct ScanRate { float log2_rate, rate; };
__device__ inline ScanRate scan_rate(float log_rate) {
  const float r = expf(log_rate);
  return {log_rate * kLog2e, r > 3e38f ? 3e38f : r};  // (a gradient times the rate is then 0, not NaN)
}
// p of a step. Below dt = -80, where exp(dt) alone would underflow, from the sum of the logarithms.
__device__ inline float scan_p(float dt, ScanRate r) {
  float e, u;
  return scan_softplus2(dt * kLog2e, e, u) * r.rate;
}
// And dp/ddt (natural) = rate sigmoid(dt).
__device__ inline float scan_p(float dt, ScanRate r, float& slope) {
  float e, u;
  const float p = scan_softplus2(dt * kLog2e, e, u) * r.rate, s = __builtin_amdgcn_rcpf(u);
  slope = (dt < 0.f ? e * s : s) * r.rate;
  return p;
}
__device__ inline float scan_p_low(float dt, ScanRate r) {
  return __builtin_amdgcn_exp2f(fmaf(dt, kLog2e, r.log2_rate)) * kLog2e;
}

// What steps, spans or a chunk make of the state h before them: u + a h, as u and the code c of their
// decay; u alone behind a reset (kScanCut). Over a span's steps the decay is the product of theirs, or
// where that is over a half, of the sum of theirs: 1 - a would be lost in the product, and the product
// in the sum (2^-p is off by p 2^-25 of itself).
constexpr float kScanCut = 2.f;
__device__ inline float scan_join(float c, float u, float h) {
  return c == kScanCut ? u : u + scan_fade(c, h);
}
// An infinite h stays infinite over any steps, as it does step by step, where its fade is NaN (h - c h, or
// 0 h where the decay of many steps underflows). Such a NaN lasts to the end of the joins or to a cut, so
// joins are walked plainly, and again with INF where the last of them is not finite (a test in each join
// cost 2.5 % of a long scan's forward, this 0 to 1).
template <bool INF>
__device__ inline float scan_join_as(float c, float u, float h) {
  return INF && c != kScanCut && !scan_finite(h) ? u + h : scan_join(c, u, h);
}
template <typename Walk>
__device__ inline float scan_joins(Walk walk, bool on = true) {
  const float h = walk(std::false_type());
  if (__builtin_expect(__any(on && !scan_finite(h)), 0)) return walk(std::true_type());
  return h;
}
// h through the spans from, from + by, .. before `to`: their codes c and u.
__device__ inline float scan_spans(int from, int to, int by, const float (*c)[64], const float (*u)[64],
                                   float h, int lane) {
  return scan_joins([&](auto inf) {
    float v = h;
    for (int w = from; w != to; w += by) v = scan_join_as<decltype(inf)::value>(c[w][lane], u[w][lane], v);
    return v;
  });
}
struct ScanDecay {
  float p = 0.f, a = 1.f;
  __device__ float code() const {
    const float w = scan_slow(p);
    return p < 1.f ? w : -a;
  }
};
// The same of joined codes.
struct ScanJoint {
  float a = 1.f, w = 0.f;
  bool cut = false;
  __device__ void then(float c) {
    cut |= c == kScanCut;
    a *= scan_a(c);
    w = fmaf(scan_w(c), 1.f - w, w);
  }
  __device__ float code() const { return cut ? kScanCut : w < 0.5f ? w : -a; }
};

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
  float *drate, *dh0;  // drate: [batch, chunks, width]
  // the states between chunks (several of them)
  uint32_t* tickets;  // [batch, tiles of the width]
  uint32_t* ends;     // [batch, groups, width]
  uint64_t* spans;    // [batch, chunks, width]
};

// ---------------------------------------------------------------------------
// The state before a chunk. Each chunk posts its span (c, u) as one 64-bit word, the last one of each
// group of kScanGroup chunks posts the state after it as one 32-bit word, and a chunk joins its
// group's earlier spans, in order, to the state that the group before it posted: always the same sums,
// whoever comes first. A word is data and flag in one: all bits set (a NaN that is never posted) is
// "not yet", and the clearing launch sets that. Workgroups take their chunk from a counter, in order
// of time, so whatever one waits for is already running; a wait that does not end in about a second
// all the same posts NaN and goes on.
// ---------------------------------------------------------------------------
constexpr uint32_t kNoWord = 0xffffffffu;
constexpr uint32_t kNanBits = 0x7fc00000u;
__device__ inline uint32_t word_of(float v) { return v == v ? __float_as_uint(v) : kNanBits; }
template <typename W>
__device__ inline void post(W* at, W v) {
  __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename W>
__device__ inline W peek(const W* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__global__ __launch_bounds__(256) void scan_clear_kernel(uint4* words, int64_t zeros, int64_t count) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t v = i < zeros ? 0 : kNoWord;
  if (i < count) words[i] = uint4{v, v, v, v};
}

// What the card holds at once, three workgroups a CU, begins over some 3 us (NAPS of 64 clocks) forward
// and 4 backward, in the order of the chain: begun together, the loads of its first chunks, for which
// all others wait, share the memory with those of its last. Walks launch after launch, their other launches
// (2.4 us forward, 6.4 backward) included, begun at once and so: forward of 16384 x 1536 54.3 and 48.8 us, 4 x
// 2048 29.3 and 25.6, 1 x 8192 34.7 and 29.9, 1 x 4096 22.2 and 19.8; backward 86.3 and 82.0, 44.7 and 43.2,
// 53.0 and 49.0, 34.8 and 31.7; 64 x 256 39.7 and 39.6. Short chains that the card holds whole begin at once:
// forward of 16 x 256 14.7, or 15.8 over 3 us.
constexpr uint32_t kScanHeld = 768;
template <uint32_t NAPS>
__device__ inline void scan_stagger(uint32_t tiles) {
  if (blockIdx.x < kScanHeld && (gridDim.x > kScanHeld || gridDim.x >= 8 * tiles))
    for (uint32_t i = blockIdx.x * NAPS / kScanHeld; i > 0; --i) __builtin_amdgcn_s_sleep(1);
}

// Which chunk (from the end where the walk starts) of which 64 channels of which sequence. Each of
// these `tiles` has a counter of its own: one for all cost 8 ns a workgroup.
struct ScanPlace { int64_t n, b, d0; };
template <bool CHAIN>
__device__ inline ScanPlace scan_place(uint32_t* tickets, int64_t width, uint32_t tiles, uint32_t* lds) {
  const uint32_t across = (uint32_t)((width + kScanLanes - 1) / kScanLanes);
  const uint32_t tile = __builtin_amdgcn_readfirstlane(blockIdx.x % tiles);
  uint32_t n = 0;
  if constexpr (CHAIN) {
    if (threadIdx.x == 0)
      *lds = __hip_atomic_fetch_add(tickets + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    n = __builtin_amdgcn_readfirstlane(*lds);
  }
  const uint32_t b = __builtin_amdgcn_readfirstlane(tile / across);
  return {n, b, (int64_t)(tile - b * across) * kScanLanes};
}

// Posts the chunk's span (c, u; wave 0's) and returns the state before it to wave 0, `first` at the
// start. The waves wait for the words side by side, and wave 0 joins them. BACK: chunks run from the
// last to the first, and place.n counts from that end.
template <int WAVES, bool BACK, typename T>
__device__ inline float scan_entry(const ScanArgs<T>& k, const ScanPlace& at, int64_t chunks,
                                   uint32_t in, bool on, int wave, float c, float u, float first,
                                   float (*words)[kScanGroup][64]) {
  constexpr int EACH = kScanGroup / WAVES;  // words of a wave: its number, + WAVES, ..
  const int lane = threadIdx.x & 63;
  const int64_t groups = (chunks + kScanGroup - 1) / kScanGroup, group = (uint32_t)at.n / kScanGroup;
  const int member = (uint32_t)at.n % kScanGroup;
  uint64_t* spans = k.spans + at.b * chunks * k.width + at.d0;
  uint32_t* ends = k.ends + at.b * groups * k.width + at.d0;
  const auto span_at = [&](int64_t n) { return spans + (BACK ? chunks - 1 - n : n) * k.width; };
  if (wave == 0 && member < kScanGroup - 1 && on)
    post(span_at(at.n) + in, ((uint64_t)word_of(c) << 32) | word_of(u));
  // The last wave has one span less (a group's last is not posted) and the end before the group.
  const bool end = wave == WAVES - 1 && group > 0;
  if (on && (wave < member || end)) {
    uint64_t w[EACH] = {};
    uint32_t e = 0;
    bool wait;
    int patience = 1 << 20;
    do {
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        if (wave + i * WAVES < member) w[i] = peek(span_at(group * kScanGroup + wave + i * WAVES) + in);
      if (end) e = peek(ends + (group - 1) * k.width + in);
      wait = e == kNoWord;
#pragma unroll
      for (int i = 0; i < EACH; ++i) wait |= w[i] == ~(uint64_t)0;
    } while (wait && --patience > 0);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      words[0][wave + i * WAVES][lane] = __uint_as_float((uint32_t)(w[i] >> 32));
      words[1][wave + i * WAVES][lane] = __uint_as_float((uint32_t)w[i]);
    }
    if (end) words[0][kScanGroup - 1][lane] = __uint_as_float(e);
  }
  __syncthreads();
  float h = first;
  if (wave == 0) {
    const float before = group > 0 ? words[0][kScanGroup - 1][lane] : first;
    h = scan_joins([&](auto inf) {
      float v = before;
      for (int m = 0; m < member; ++m)
        v = scan_join_as<decltype(inf)::value>(words[0][m][lane], words[1][m][lane], v);
      return v;
    }, on);
    if (member == kScanGroup - 1 && on)
      post(ends + group * k.width + in, word_of(scan_join_as<true>(c, u, h)));
  }
  return h;
}

// A row that all lanes share, in two scalar registers, from which a lane reads or writes at its byte
// offset (made anew for each access: widened to 64 bits once for all, it costs a sum in every lane for
// each). next() keeps it a running pointer: left alone, the compiler computes all rows' addresses
// ahead and spills them.
// STREAM: past the caches (scan_stream).
template <typename T, bool STREAM = false>
struct ScanRow {
  using Raw = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
  using Global = __attribute__((address_space(1))) char*;
  Global at;
  int64_t by;
  __device__ ScanRow(const T* p, int64_t step) : at((Global)(char*)p), by(step * (int64_t)sizeof(T)) {}
  __device__ T load(uint32_t off) const {
    asm("" : "+v"(off));
    const auto p = (__attribute__((address_space(1))) Raw*)(at + off);
    return __builtin_bit_cast(T, STREAM ? __builtin_nontemporal_load(p) : *p);
  }
  __device__ void store(uint32_t off, float v) const {
    asm("" : "+v"(off));
    const auto p = (__attribute__((address_space(1))) Raw*)(at + off);
    const Raw raw = __builtin_bit_cast(Raw, io<T>::from_f32(v));
    if constexpr (STREAM) __builtin_nontemporal_store(raw, p);
    else *p = raw;
  }
  __device__ void next(bool there = true) {  // (else the same row again)
    at += there ? by : 0;
    asm volatile("" : "+s"(at));
  }
};

// Every four steps the compiler may not mix with later ones: enough to overlap, and registers for three
// workgroups a CU.
__device__ inline void scan_pace(int i) {
  if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
}

// The resets of a span's steps as bits (bit i: step i).
__device__ inline uint32_t scan_resets(const uint8_t* reset, int64_t row, int n) {
  const int lane = threadIdx.x & 63;
  const bool cut = reset && lane < n && reset[row + lane];
  return __builtin_amdgcn_readfirstlane((uint32_t)__ballot(cut));
}

// Forward: a workgroup takes one chunk of 64 channels.
template <typename T, bool CHAIN, int STREAM = 0>
__global__ __launch_bounds__(64 * kScanWaves, 6) void gated_scan_fwd_kernel(ScanArgs<T> k, uint32_t tiles) {
  __shared__ float part[2][kScanWaves][64];  // c and u of each span
  __shared__ float words[CHAIN ? 2 : 1][kScanGroup][64], entry[64];
  __shared__ uint32_t place;
  using In = ScanRow<T, STREAM == 2>;
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if constexpr (CHAIN) scan_stagger<96>(tiles);
  const ScanPlace at = scan_place<CHAIN>(k.tickets, k.width, tiles, &place);
  const int64_t d = at.d0 + lane, b = at.b;
  const bool on = d < k.width;
  const uint32_t in = on ? lane : (uint32_t)(k.width - 1 - at.d0);  // lanes past the end read the last
  const int64_t dc = at.d0 + in;
  const uint32_t off = in * (uint32_t)sizeof(T);
  const int64_t chunk = (int64_t)waves * kScanSteps, chunks = CHAIN ? (k.seq + chunk - 1) / chunk : 1;
  const int64_t t0 = at.n * chunk + wave * kScanSteps, row0 = b * k.seq + t0;
  const int n = k.seq - t0 < kScanSteps ? (k.seq > t0 ? (int)(k.seq - t0) : 0) : kScanSteps;
  const ScanRate rate = scan_rate(k.log_rate[dc]);
  float a[kScanSteps], ws[kScanSteps];  // h = a h + ws; a is p at first
  const uint32_t cuts = scan_resets(k.reset, row0, n);
  ScanDecay decay;
  float u = 0.f;
  // PLAIN: all steps are there and none is a reset.
  const auto walk = [&](auto plain) {
    constexpr bool PLAIN = decltype(plain)::value;
    In dts(k.dt + row0 * k.dt_row + at.d0, k.dt_row);
    In gs(k.g + row0 * k.g_row + at.d0, k.g_row), xs(k.x + row0 * k.x_row + at.d0, k.x_row);
    T raw[3][kScanSteps];
#pragma unroll
    for (int i = 0; i < kScanSteps; ++i) {
      raw[0][i] = dts.load(off);
      dts.next(PLAIN || i + 1 < n);
    }
#pragma unroll
    for (int i = 0; i < kScanSteps; ++i) {
      raw[1][i] = gs.load(off), raw[2][i] = xs.load(off);
      gs.next(PLAIN || i + 1 < n), xs.next(PLAIN || i + 1 < n);
    }
    __builtin_amdgcn_sched_barrier(0);  // all loads first
    float low = 0.f;
#pragma unroll
    for (int i = 0; i < kScanSteps; ++i) {
      const float dt = io<T>::to_f32(raw[0][i]);
      low = fminf(low, dt);
      a[i] = scan_p(dt, rate);
      scan_pace(i);
    }
    if (__builtin_expect(__any(low < -80.f), 0)) {
      In again(k.dt + row0 * k.dt_row + at.d0, k.dt_row);
#pragma unroll
      for (int i = 0; i < kScanSteps; ++i) {
        const float dt = io<T>::to_f32(again.load(off));
        again.next(PLAIN || i + 1 < n);
        if (dt < -80.f) a[i] = scan_p_low(dt, rate);
      }
    }
#pragma unroll
    for (int i = 0; i < kScanSteps; ++i) {
      const float gate = __builtin_amdgcn_rcpf(1.f + __expf(-io<T>::to_f32(raw[1][i])));
      float s = io<T>::to_f32(raw[2][i]) * gate, p = a[i], w;
      if (!PLAIN) {
        if (i >= n) p = s = 0.f;  // a step that changes nothing
        if (cuts >> i & 1) u = 0.f;
      }
      scan_pair(p, a[i], w);
      ws[i] = w * s;
      decay.p += p;
      decay.a *= a[i];
      u = fmaf(a[i], u, ws[i]);
      scan_pace(i);
    }
  };
  const bool plain = n == kScanSteps && cuts == 0;
  if (plain) walk(std::true_type());
  else if (n > 0) walk(std::false_type());
  part[0][wave][lane] = cuts ? kScanCut : decay.code();
  part[1][wave][lane] = u;
  float h = 0.f;
  if (wave == 0 && at.n == 0) {
    h = k.h0 ? k.h0[b * k.width + dc] : 0.f;
    entry[lane] = h;
  }
  __syncthreads();
  if constexpr (CHAIN) {
    float cu = 0.f, cc = 0.f;
    if (wave == 0) {
      ScanJoint all;
      all.cut = at.n == 0;  // the first chunk posts its state (h0 is not read again: h_last may be h0)
#pragma unroll
      for (int w = 0; w < kScanWaves; ++w) all.then(part[0][w][lane]);
      cu = scan_joins([&](auto inf) {
        float v = h;
#pragma unroll
        for (int w = 0; w < kScanWaves; ++w)
          v = scan_join_as<decltype(inf)::value>(part[0][w][lane], part[1][w][lane], v);
        return v;
      });
      cc = all.code();
    }
    h = scan_entry<kScanWaves, false>(k, at, chunks, in, on, wave, cc, cu, h, words);
    if (wave == 0) entry[lane] = h;
    __syncthreads();
  }
  h = entry[lane];
  if (n == 0) {
    if (k.seq == 0 && k.h_last && on && wave == 0) k.h_last[b * k.width + d] = h;
    return;
  }
  h = scan_spans(0, wave, 1, part[0], part[1], h, lane);
  if (k.carries && t0 % kScanChunk == 0 && on) {
    const int64_t every = (k.seq + kScanChunk - 1) / kScanChunk;
    k.carries[(b * every + t0 / kScanChunk) * k.width + d] = h;
  }
  if (!on) return;
  ScanRow<T, (STREAM > 0)> y(k.y + row0 * k.width + at.d0, k.width);
  if (plain) {
#pragma unroll
    for (int i = 0; i < kScanSteps; ++i) {
      h = fmaf(a[i], h, ws[i]);
      y.store(off, h);
      y.next();
    }
  } else {
#pragma unroll
    for (int i = 0; i < kScanSteps; ++i)
      if (i < n) {
        if (cuts >> i & 1) h = 0.f;
        h = fmaf(a[i], h, ws[i]);
        y.store(off, h);
        y.next();
      }
  }
  if (k.h_last && t0 + n == k.seq) k.h_last[b * k.width + d] = h;
}

// Backward: the chunks from the last to the first, each from its stored entry state. What a span makes
// of the adjoint A behind it (A = a G of the step after) is v + 2^-p A.
template <typename T, bool CHAIN, int STREAM = 0>
__global__ __launch_bounds__(64 * kBackWaves) void gated_scan_bwd_kernel(ScanArgs<T> k, uint32_t tiles) {
  __shared__ float part[3][kBackWaves][64];  // c, u and v of each span
  __shared__ float words[CHAIN ? 2 : 1][kScanGroup][64], entry[64];
  __shared__ uint32_t place;
  using In = ScanRow<T, STREAM == 2>;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if constexpr (CHAIN) scan_stagger<128>(tiles);
  const ScanPlace at = scan_place<CHAIN>(k.tickets, k.width, tiles, &place);
  const int64_t d = at.d0 + lane, b = at.b;
  const bool on = d < k.width;
  const uint32_t in = on ? lane : (uint32_t)(k.width - 1 - at.d0);  // lanes past the end read the last
  const int64_t dc = at.d0 + in;
  const uint32_t off = in * (uint32_t)sizeof(T);
  const int64_t chunks = CHAIN ? (k.seq + kScanChunk - 1) / kScanChunk : 1, j = chunks - 1 - at.n;
  const int64_t t0 = j * kScanChunk + wave * kBackSteps, row0 = b * k.seq + t0;
  const int n = k.seq - t0 < kBackSteps ? (k.seq > t0 ? (int)(k.seq - t0) : 0) : kBackSteps;
  const ScanRate rate = scan_rate(k.log_rate[dc]);
  // a; s, later s - h; dy; w = 1 - a; sigmoid(g); s (1 - sigmoid(g)); dp/ddt = rate sigmoid(dt); p
  float a[kBackSteps], e[kBackSteps], dy[kBackSteps], w[kBackSteps], sg[kBackSteps], q[kBackSteps],
      sd[kBackSteps], ps[kBackSteps];
  const uint32_t cuts = scan_resets(k.reset, row0, n);
  ScanDecay decay;
  float u = 0.f, v = 0.f;
  // PLAIN: all steps are there and none is a reset.
  const auto walk = [&](auto plain) {
    constexpr bool PLAIN = decltype(plain)::value;
    In dts(k.dt + row0 * k.dt_row + at.d0, k.dt_row);
    In gs(k.g + row0 * k.g_row + at.d0, k.g_row), xs(k.x + row0 * k.x_row + at.d0, k.x_row);
    In dys(k.dy + row0 * k.width + at.d0, k.width);
    T raw[4][kBackSteps];
#pragma unroll
    for (int i = 0; i < kBackSteps; ++i) {
      raw[0][i] = dts.load(off);
      dts.next(PLAIN || i + 1 < n);
    }
#pragma unroll
    for (int i = 0; i < kBackSteps; ++i) {
      raw[1][i] = gs.load(off), raw[2][i] = xs.load(off), raw[3][i] = dys.load(off);
      gs.next(PLAIN || i + 1 < n), xs.next(PLAIN || i + 1 < n), dys.next(PLAIN || i + 1 < n);
    }
    __builtin_amdgcn_sched_barrier(0);  // all loads first
    float low = 0.f;
#pragma unroll
    for (int i = 0; i < kBackSteps; ++i) {
      const float dt = io<T>::to_f32(raw[0][i]);
      low = fminf(low, dt);
      ps[i] = scan_p(dt, rate, sd[i]);
      scan_pace(i);
    }
    if (__builtin_expect(__any(low < -80.f), 0)) {
      In again(k.dt + row0 * k.dt_row + at.d0, k.dt_row);
#pragma unroll
      for (int i = 0; i < kBackSteps; ++i) {
        const float dt = io<T>::to_f32(again.load(off));
        again.next(PLAIN || i + 1 < n);
        if (dt < -80.f) ps[i] = scan_p_low(dt, rate), sd[i] = ps[i] * kLn2;
      }
    }
#pragma unroll
    for (int i = 0; i < kBackSteps; ++i) {
      float cg;
      sigmoid_pair(io<T>::to_f32(raw[1][i]), sg[i], cg);
      e[i] = io<T>::to_f32(raw[2][i]) * sg[i];
      q[i] = e[i] * cg;
      dy[i] = io<T>::to_f32(raw[3][i]);
      if (!PLAIN) {
        if (i >= n) ps[i] = e[i] = dy[i] = 0.f;  // a step that changes nothing
        if (cuts >> i & 1) u = 0.f;
      }
      scan_pair(ps[i], a[i], w[i]);
      decay.p += ps[i];
      decay.a *= a[i];
      u = fmaf(a[i], u, w[i] * e[i]);
      scan_pace(i);
    }
#pragma unroll
    for (int i = kBackSteps - 1; i >= 0; --i)
      v = !PLAIN && (cuts >> i & 1) ? 0.f : a[i] * (dy[i] + v);
  };
  const bool all = n == kBackSteps && cuts == 0;
  if (all) walk(std::true_type());
  else if (n > 0) walk(std::false_type());
  part[0][wave][lane] = cuts ? kScanCut : decay.code();
  part[1][wave][lane] = u;
  part[2][wave][lane] = v;
  __syncthreads();
  float A = k.dh_last ? k.dh_last[b * k.width + dc] : 0.f;
  if constexpr (CHAIN) {
    float cv = 0.f, cc = 0.f;
    if (wave == 0) {
      ScanJoint all;
#pragma unroll
      for (int w = kBackWaves - 1; w >= 0; --w) all.then(part[0][w][lane]);
      cv = scan_joins([&](auto inf) {
        float v = 0.f;
#pragma unroll
        for (int w = kBackWaves - 1; w >= 0; --w)
          v = scan_join_as<decltype(inf)::value>(part[0][w][lane], part[2][w][lane], v);
        return v;
      });
      cc = all.code();
    }
    A = scan_entry<kBackWaves, true>(k, at, chunks, in, on, wave, cc, cv, A, words);
    if (wave == 0) entry[lane] = A;
    __syncthreads();
    A = entry[lane];
  }
  float drate = 0.f;
  if (n > 0) {
    float h = k.carries[(b * chunks + j) * k.width + dc];
    h = scan_spans(0, wave, 1, part[0], part[1], h, lane);
    A = scan_spans(kBackWaves - 1, wave, -1, part[0], part[2], A, lane);
    const auto back = [&](auto plain) {
      constexpr bool PLAIN = decltype(plain)::value;
#pragma unroll
      for (int i = 0; i < kBackSteps; ++i)
        if (PLAIN || i < n) {
          if (!PLAIN && (cuts >> i & 1)) h = 0.f;
          const float s = e[i];
          e[i] = s - h;
          h = fmaf(a[i], h, w[i] * s);
        }
      const int64_t to = (row0 + (PLAIN ? kBackSteps : n) - 1) * k.width + at.d0;
      ScanRow<T, (STREAM > 0)> ddt(k.ddt + to, -k.width), dg(k.dg + to, -k.width), dx(k.dx + to, -k.width);
#pragma unroll
      for (int i = kBackSteps - 1; i >= 0; --i)
        if (PLAIN || i < n) {
          const float G = dy[i] + A, aG = a[i] * G;
          const float dp = aG * e[i], ds = w[i] * G;
          ddt.store(off, dp * sd[i]);
          dg.store(off, ds * q[i]);
          dx.store(off, ds * sg[i]);
          ddt.next(), dg.next(), dx.next();
          // (2^-p is 0 long before p = 300: no 0 times infinity)
          drate = fmaf(dp, fminf(ps[i], 300.f), drate);
          A = !PLAIN && (cuts >> i & 1) ? 0.f : aG;
        }
    };
    if (on) {
      if (all) back(std::true_type());
      else back(std::false_type());
    }
    if (k.dh0 && on && t0 == 0) k.dh0[b * k.width + d] = A;
  }
  __syncthreads();
  part[0][wave][lane] = drate;
  __syncthreads();
  if (wave == 0 && on) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kBackWaves; ++w) sum += part[0][w][lane];
    k.drate[(b * chunks + j) * k.width + d] = sum * kLn2;
  }
}

// One token for each sequence, the state in place. 16 x 1536 in fp16 3 us, a launch's latency (7 with
// the host).
template <typename T>
__global__ __launch_bounds__(256) void gated_scan_step_kernel(ScanArgs<T> k, float* h) {
  const int64_t d = (int64_t)blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
  if (d >= k.width) return;
  const float dt = load_scalar(k.dt + b * k.dt_row + d), g = load_scalar(k.g + b * k.g_row + d);
  const float s = load_scalar(k.x + b * k.x_row + d) * __builtin_amdgcn_rcpf(1.f + __expf(-g));
  const ScanRate rate = scan_rate(k.log_rate[d]);
  const float p = dt < -80.f ? scan_p_low(dt, rate) : scan_p(dt, rate), old = h[b * k.width + d];
  float a, w;
  scan_pair(p, a, w);
  // Away from whichever is the larger part: an a near 1, rounded, would leave its mark at each token.
  float v = p < 1.f ? fmaf(w, s - old, old) : fmaf(a, old - s, s);
  if (!scan_finite(v)) v = fmaf(a, old, w * s);  // infinities do not meet their negatives
  h[b * k.width + d] = v;
  store_scalar(k.y + b * k.width + d, v);
}

// The workspace of a launch over several chunks: the tiles' counters, the spans, the ends (each from a
// multiple of 16 bytes); and of the backward the partial sums of dlog_rate behind them.
struct ScanSpace { int64_t chunks, counters, spans, bytes; };
inline ScanSpace scan_space(int64_t batch, int64_t seq, int64_t width, int64_t chunk) {
  const int64_t chunks = (seq + chunk - 1) / chunk, groups = (chunks + kScanGroup - 1) / kScanGroup;
  if (chunks <= 1) return {chunks, 0, 0, 0};
  const auto whole = [](int64_t bytes) { return (bytes + 15) / 16 * 16; };
  const int64_t counters = whole(4 * batch * ((width + kScanLanes - 1) / kScanLanes));
  const int64_t spans = whole(8 * batch * chunks * width);
  return {chunks, counters, spans, counters + spans + whole(4 * batch * groups * width)};
}

template <typename T>
int scan_chain(ScanArgs<T>& k, const ScanSpace& w, char* ws, hipStream_t s) {
  k.tickets = (uint32_t*)ws;
  k.spans = (uint64_t*)(ws + w.counters);
  k.ends = (uint32_t*)(ws + w.counters + w.spans);
  const int64_t quads = w.bytes / 16;
  scan_clear_kernel<<<dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s>>>(
      (uint4*)ws, w.counters / 16, quads);
  return launch_status();
}

// What the 256 MiB cache does not hold anyway goes past it: the outputs where they and the inputs are
// more, the inputs where these alone are. bf16, launch after launch with their other launches: backward of 8
// x 2048 x 1536 (201 MB in, 151 out) 97.5 us, with outputs streamed 73.5, with both 92.7; 1 x 65536 forward
// 209.8, 204.8, 200.4, backward 405, 392, 375; what fits gains little or loses, and whoever reads its outputs
// next finds them in the cache: 4 x 2048 forward 25.7, 25.4, 27.5, backward 43.2, 42.2, 52.5.
inline int scan_stream(int64_t tensor, int in, int out) {
  return tensor * in > (256LL << 20) ? 2 : tensor * (in + out) > (256LL << 20) ? 1 : 0;
}
#define MQC_SCAN_CHAIN(KERNEL, WAVES, IN, OUT)                                                        \
  const dim3 grid((unsigned)(tiles * w.chunks)), block(64 * WAVES);                                   \
  switch (scan_stream(batch * k.seq * k.width * (int64_t)sizeof(T), IN, OUT)) {                       \
    case 0: KERNEL<T, true, 0><<<grid, block, 0, s>>>(k, (uint32_t)tiles); break;                     \
    case 1: KERNEL<T, true, 1><<<grid, block, 0, s>>>(k, (uint32_t)tiles); break;                     \
    default: KERNEL<T, true, 2><<<grid, block, 0, s>>>(k, (uint32_t)tiles); break;                    \
  }

// A forward's waves of a workgroup: those that have steps.
inline int scan_waves(int64_t seq) {
  return seq > kScanWaves * kScanSteps ? kScanWaves : seq > 0 ? (int)((seq + kScanSteps - 1) / kScanSteps) : 1;
}
template <typename T>
int launch_gated_scan_fwd(ScanArgs<T> k, int64_t batch, char* ws, hipStream_t s) {
  const int64_t tiles = batch * ((k.width + kScanLanes - 1) / kScanLanes);
  const ScanSpace w = scan_space(batch, k.seq, k.width, kScanWaves * kScanSteps);
  if (w.chunks > 1) {
    const int st = scan_chain(k, w, ws, s);
    if (st != MQC_OK) return st;
    MQC_SCAN_CHAIN(gated_scan_fwd_kernel, kScanWaves, 3, 1)
  } else {
    gated_scan_fwd_kernel<T, false>
        <<<dim3((unsigned)tiles), dim3(64 * (unsigned)scan_waves(k.seq)), 0, s>>>(k, (uint32_t)tiles);
  }
  return launch_status();
}

template <typename T>
int launch_gated_scan_bwd(ScanArgs<T> k, int64_t batch, float* drate, char* ws, hipStream_t s) {
  const int64_t tiles = batch * ((k.width + kScanLanes - 1) / kScanLanes);
  const ScanSpace w = scan_space(batch, k.seq, k.width, kScanChunk);
  k.drate = (float*)(ws + w.bytes);
  if (w.chunks > 1) {
    const int st = scan_chain(k, w, ws, s);
    if (st != MQC_OK) return st;
    MQC_SCAN_CHAIN(gated_scan_bwd_kernel, kBackWaves, 4, 3)
  } else {
    gated_scan_bwd_kernel<T, false>
        <<<dim3((unsigned)tiles), dim3(64 * kBackWaves), 0, s>>>(k, (uint32_t)tiles);
  }
  const int st = launch_status();
  if (st != MQC_OK) return st;
  return mqc_sum_rows(k.drate, drate, k.width, nullptr, nullptr, 0, nullptr, nullptr, 0,
                      batch * w.chunks, s);
}
#undef MQC_SCAN_CHAIN

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
// Whether a walk is one launch: 2^36 elements, and of narrow tensors fewer (a width of 1 takes the
// workgroups of 64).
inline bool scan_fits(int64_t batch, int64_t seq, int64_t width, int waves) {
  const int64_t chunk = waves * kScanSteps, chunks = seq > chunk ? (seq + chunk - 1) / chunk : 1;
  const int64_t tiles = batch * ((width + kScanLanes - 1) / kScanLanes);  // below 2^42
  return launchable(tiles, 64 * waves) && launchable(tiles * chunks, 64 * waves);
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
  const ScanSpace w = scan_space(batch, seq_len, width, kScanChunk);
  return w.bytes + batch * w.chunks * width * (int64_t)sizeof(float);
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
  if (!scan_fits(batch, seq_len, width, scan_waves(seq_len))) return MQC_E_LIMIT;
  if (!log_rate || (seq_len > 0 && (!dt || !g || !x || !y))) return MQC_E_NULL;
  if (seq_len == 0 && !h_last) return MQC_OK;
  if (workspace_bytes < mqc_gated_scan_workspace_bytes(batch, seq_len, width)) return MQC_E_SPACE;
  if (workspace_bytes > 0 && !workspace) return MQC_E_NULL;
  if (!aligned(workspace, 16)) return MQC_E_ALIGN;
#define MQC_F(T)                                                                               \
  [&] {                                                                                        \
    ScanArgs<T> k = scan_args<T>(dt, dt_row, g, g_row, x, x_row, log_rate, reset, seq_len, width); \
    k.h0 = h0; k.y = (T*)y; k.h_last = h_last; k.carries = carries;                            \
    return launch_gated_scan_fwd<T>(k, batch, (char*)workspace, (hipStream_t)stream);                            \
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
  if (!scan_fits(batch, seq_len, width, kBackWaves)) return MQC_E_LIMIT;
  if (!dt || !g || !x || !log_rate || !carries || !dy || !ddt || !dg || !dx || !dlog_rate ||
      !workspace)
    return MQC_E_NULL;
  if (workspace_bytes < mqc_gated_scan_workspace_bytes(batch, seq_len, width)) return MQC_E_SPACE;
  if (!aligned(workspace, 16)) return MQC_E_ALIGN;
#define MQC_F(T)                                                                               \
  [&] {                                                                                        \
    ScanArgs<T> k = scan_args<T>(dt, dt_row, g, g_row, x, x_row, log_rate, reset, seq_len, width); \
    k.carries = const_cast<float*>(carries);                                                   \
    k.dy = (const T*)dy; k.dh_last = dh_last; k.ddt = (T*)ddt; k.dg = (T*)dg; k.dx = (T*)dx;    \
    k.dh0 = dh0;                                                                               \
    return launch_gated_scan_bwd<T>(k, batch, dlog_rate, (char*)workspace, (hipStream_t)stream); \
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
