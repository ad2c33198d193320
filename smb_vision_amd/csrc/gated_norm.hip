// The norm behind a block, its gate, the scaled residual sum and the norm in front of the next block as one pass, and its gradient:
//     n = post(h) = hhat post_w + post_b,   x1 = res_scale x + gate n,   y = pre(x1) = xhat pre_w + pre_b
// with hhat = (h - mean) / deviation (RMS norm: mean 0), the gate one row for `rows_per_gate` consecutive rows, and
//     t  = dx1 + pre^T(dy),   dx = res_scale t,   dgate = sum t n,   dh = post^T(gate t),   dpost_w = sum gate t hhat,  dpre_w = sum dy xhat, ...
//     norm^T(g) with z = w g:  (z - [LayerNorm: mean z] - hat mean(z hat)) / deviation
// Bound by HBM: the forward reads h, x and writes x1, y; the backward reads dx1, dy, h, x (x1 is formed again from h and x in 32 bits rather than read back
// rounded) and writes dh, dx.  A row lives in the registers of K waves, 8 elements a lane (12 where that spares a second wave: 768): what the backward keeps
// beside a row - three parameters and four sums a column - then leaves four waves a SIMD (with 16 a lane it spilled: 184 us instead of 64 at 20,480 x 768).
// (20,480 x 768, h in bf16 and x in fp32: forward 36 us, 5.2 TB/s; backward 63 us, 4.5 TB/s; its sums 8.)  A workgroup walks rows with the parameters in registers.  Sums and statistics are fp32, variances about the mean.
// The parameters' gradients: every workgroup owns a run of rows and adds its rows' terms in registers; a second launch adds the workgroups' sums in a fixed
// order (no float atomics: the result repeats bit for bit).  Within a gate's rows sum t n = post_w sum t hhat + post_b sum t, and the same two sums times the gate
// are dpost_w and dpost_b.
#include "smbv_common.h"
#include "smbv_kernels.h"
#include <math.h>

namespace smbv {

// V elements of a row at once.  WIDE: rows start on 16 bytes and end on a whole vector; otherwise the vectors are read where they lie (the memory takes any
// alignment) and the row's last d % V elements, one to a lane, are a register more.  (One lane that took them one after the other: 25.9 us instead of 18.2
// for the forward of 7108 x 1004 in bf16, where four are left.)
template <class T, int V, bool WIDE> struct __attribute__((packed, aligned(WIDE ? (sizeof(T) * V > 16 ? 16 : sizeof(T) * V) : sizeof(T)))) GnVec { T e[V]; };

// the row's elements of this lane: NE of them in vectors of V, vector i at column (i LANES + lane) V, and one behind the vectors; past the row's end zeros
template <class T, int NE, int V, int LANES, bool WIDE>
__device__ __forceinline__ void gn_load(float (&f)[NE + !WIDE], const T* p, int lane, int d, bool on) {
#pragma unroll
  for (int i = 0; i < NE / V; i++) {
    const int c = (i * LANES + lane) * V;
    if (on && c + V <= d) {
      const GnVec<T, V, WIDE> v = *(const GnVec<T, V, WIDE>*)(p + c);
#pragma unroll
      for (int e = 0; e < V; e++) f[i * V + e] = (float)v.e[e];
    } else {
#pragma unroll
      for (int e = 0; e < V; e++) f[i * V + e] = 0.f;
    }
  }
  if constexpr (!WIDE) f[NE] = on && lane < d % V ? (float)p[d - d % V + lane] : 0.f;
}
template <class T, int NE, int V, int LANES, bool WIDE>
__device__ __forceinline__ void gn_store(const float (&f)[NE + !WIDE], T* p, int lane, int d) {
#pragma unroll
  for (int i = 0; i < NE / V; i++) {
    const int c = (i * LANES + lane) * V;
    if (c + V <= d) {
      GnVec<T, V, WIDE> v;
#pragma unroll
      for (int e = 0; e < V; e++) v.e[e] = (T)f[i * V + e];
      *(GnVec<T, V, WIDE>*)(p + c) = v;
    }
  }
  if constexpr (!WIDE) {
    if (lane < d % V) p[d - d % V + lane] = (T)f[NE];
  }
}
template <int NE, int V, int LANES, bool WIDE>
__device__ __forceinline__ void gn_param(float (&f)[NE + !WIDE], const float* p, float none, int lane, int d) {
  if (p) gn_load<float, NE, V, LANES, WIDE>(f, p, lane, d, true);
  else {
#pragma unroll
    for (int i = 0; i < NE + !WIDE; i++) f[i] = none;
  }
}
// is register i of this lane inside the row
template <int NE, int V, int LANES> __device__ __forceinline__ bool gn_in(int i, int lane, int d) {
  return i < NE ? ((i / V) * LANES + lane) * V + V <= d : lane < d % V;
}

// sums over a row's K waves; every wave of the workgroup calls it the same number of times (two alternating slots: one barrier a call)
template <int K, int WAVES>
struct GnReduce {
  float* slots;  // LDS [2][waves][2]
  int flip;
  template <int N>
  __device__ __forceinline__ void operator()(float (&s)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) s[i] = wave_sum(s[i]);
    if constexpr (K > 1) {
      const int w = threadIdx.x >> 6, l = threadIdx.x & 63, w0 = w & ~(K - 1);
      float* at = slots + flip * WAVES * 2;
      if (l == 0) {
#pragma unroll
        for (int i = 0; i < N; i++) at[w * 2 + i] = s[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; i++) {
        s[i] = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) s[i] += at[(w0 + k) * 2 + i];
      }
      flip ^= 1;
    }
  }
};

template <int NE, int V, int LANES, bool WIDE, class R>
__device__ __forceinline__ void gn_stats(const float (&f)[NE + !WIDE], int kind, int lane, int d, float eps, float& mu, float& rs, R& red) {
  constexpr int N = NE + !WIDE;
  mu = 0.f;
  if (kind == 2) {
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < N; i++) s[0] += f[i];
    red(s);
    mu = s[0] / d;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float c = gn_in<NE, V, LANES>(i, lane, d) ? f[i] - mu : 0.f;
    q[0] += c * c;
  }
  red(q);
  rs = 1.0f / sqrtf(q[0] / d + eps);
}

// a workgroup has 4 waves, or the 8 or 16 that one row takes
template <class TH, class TX, int NE, int V, int K, bool WIDE>
__global__ __launch_bounds__(K > 4 ? 64 * K : 256) void gated_norm_fwd_kernel(GatedNormDesc d) {
  constexpr int LANES = 64 * K, WAVES = K > 4 ? K : 4, TEAMS = WAVES / K, N = NE + !WIDE;
  __shared__ float slots[2 * WAVES * 2];
  const int lane = threadIdx.x & (LANES - 1), team = __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
  GnReduce<K, WAVES> red{slots, 0};
  float w[N], b[N], gt[N], pw[N], pb[N];
  gn_param<NE, V, LANES, WIDE>(w, d.post_w, 1.f, lane, d.d);
  gn_param<NE, V, LANES, WIDE>(b, d.post_b, 0.f, lane, d.d);
  gn_param<NE, V, LANES, WIDE>(pw, d.pre_w, 1.f, lane, d.d);
  gn_param<NE, V, LANES, WIDE>(pb, d.pre_b, 0.f, lane, d.d);
  gn_param<NE, V, LANES, WIDE>(gt, nullptr, 1.f, lane, d.d);
  long long g = -1;
  for (long long base = (long long)blockIdx.x * TEAMS; base < d.rows; base += (long long)gridDim.x * TEAMS) {
    const long long row = base + team;
    const bool on = row < d.rows;
    float h[N], x[N];
    gn_load<TH, NE, V, LANES, WIDE>(h, (const TH*)d.h + row * d.ldh, lane, d.d, on);
    gn_load<TX, NE, V, LANES, WIDE>(x, (const TX*)d.x + row * d.ldx, lane, d.d, on);
    if (d.gate && on && row / d.rows_per_gate != g) {
      g = row / d.rows_per_gate;
      gn_load<float, NE, V, LANES, WIDE>(gt, d.gate + g * d.d, lane, d.d, true);
    }
    float mu = 0.f, rs = 1.f;
    if (d.post) {
      gn_stats<NE, V, LANES, WIDE>(h, d.post, lane, d.d, d.eps, mu, rs, red);
#pragma unroll
      for (int i = 0; i < N; i++) h[i] = (h[i] - mu) * rs * w[i] + b[i];
    }
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = gn_in<NE, V, LANES>(i, lane, d.d) ? __builtin_fmaf(d.res_scale, x[i], h[i] * gt[i]) : 0.f;
    if (on) gn_store<TX, NE, V, LANES, WIDE>(x, (TX*)d.x1 + row * d.ldx1, lane, d.d);
    float mx = 0.f, rx = 1.f;
    if (d.pre) {
      gn_stats<NE, V, LANES, WIDE>(x, d.pre, lane, d.d, d.eps, mx, rx, red);
#pragma unroll
      for (int i = 0; i < N; i++) x[i] = (x[i] - mx) * rx * pw[i] + pb[i];
      if (on) gn_store<TH, NE, V, LANES, WIDE>(x, (TH*)d.y + row * d.ldy, lane, d.d);
    }
    if (on && lane == 0) *(f32x4*)(d.stats + 4 * row) = (f32x4){mu, rs, mx, rx};
  }
}

// workspace of the backward: sums of C workgroups, [C][d] each: pre_w | pre_b | post_w | post_b, then [C][2][d]: of the gates that a workgroup shares with others -
// the one that its rows begin with, and the one that begins inside them and goes on behind them
struct GnPart { float* base; int C; long long chunk; };

// Four waves a SIMD where the registers go round: three with 12 elements a lane, or with the register for a row's last elements (four: 20 spilled, 40 us
// instead of 32 at 7108 x 1001) - but not with 8 waves a row, of whose workgroups three waves a SIMD hold one instead of two (7108 x 4001: 154 us instead of 131)
template <class TH, class TX, int NE, int V, int K, bool WIDE, bool PER_ROW>
__global__ __launch_bounds__(K > 4 ? 64 * K : 256) __attribute__((amdgpu_waves_per_eu(NE > 8 || (!WIDE && K < 8) ? 3 : 4))) void gated_norm_bwd_kernel(GatedNormDesc d, GnPart part) {
  constexpr int LANES = 64 * K, WAVES = K > 4 ? K : 4, TEAMS = WAVES / K, N = NE + !WIDE;
  __shared__ float slots[2 * WAVES * 2];
  __shared__ float fold[2 * N * 64 * WAVES];   // the teams' sums on their way out; between a workgroup's runs of rows: its sums for post_w, post_b
  const int tid = threadIdx.x, lane = tid & (LANES - 1), team = __builtin_amdgcn_readfirstlane(tid / LANES);
  GnReduce<K, WAVES> red{slots, 0};
  const long long c0 = blockIdx.x * part.chunk, c1 = c0 + part.chunk < d.rows ? c0 + part.chunk : d.rows;
  float sw[N], sb[N], pw[N];   // sums for pre_w, pre_b
#pragma unroll
  for (int i = 0; i < N; i++) { sw[i] = 0.f; sb[i] = 0.f; fold[i * 64 * WAVES + tid] = 0.f; fold[(N + i) * 64 * WAVES + tid] = 0.f; }
  gn_param<NE, V, LANES, WIDE>(pw, d.pre_w, 1.f, lane, d.d);
  // the teams' sums of a column, in their order, and out by team 0
  auto flush = [&](float (&s)[N], float* out) __attribute__((always_inline)) {
    if constexpr (TEAMS > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; i++) fold[i * 64 * WAVES + tid] = s[i];
      __syncthreads();
      if (team == 0) {
        for (int k = 1; k < TEAMS; k++)
#pragma unroll
          for (int i = 0; i < N; i++) s[i] += fold[i * 64 * WAVES + k * LANES + lane];
      }
    }
    if (team == 0) gn_store<float, NE, V, LANES, WIDE>(s, out, lane, d.d);
  };
  const bool gated = d.gate && !PER_ROW;
  const long long rpg = gated ? d.rows_per_gate : d.rows;
  for (long long s0 = c0; s0 < c1;) {   // runs of rows with one gate
    const long long g = s0 / rpg, s1 = (g + 1) * rpg < c1 ? (g + 1) * rpg : c1;
    float gw[N], gb[N], sa[N], sc[N];   // gate post_w, gate post_b; sums of t hhat and t over these rows
    {
      float w[N];
      gn_param<NE, V, LANES, WIDE>(gw, gated ? d.gate + g * d.d : nullptr, 1.f, lane, d.d);
      gn_param<NE, V, LANES, WIDE>(gb, d.post_b, 0.f, lane, d.d);
      gn_param<NE, V, LANES, WIDE>(w, d.post_w, 1.f, lane, d.d);
#pragma unroll
      for (int i = 0; i < N; i++) { gb[i] *= gw[i]; gw[i] *= w[i]; sa[i] = 0.f; sc[i] = 0.f; }
    }
    for (long long base = s0; base < s1; base += TEAMS) {
      const long long row = base + team;
      const bool on = row < s1;
      f32x4 st = {0.f, 0.f, 0.f, 0.f};
      if (on) st = *(const f32x4*)(d.stats + 4 * row);
      float h[N], x[N], t[N], dy[N], gr[PER_ROW ? N : 1];
      gn_load<TH, NE, V, LANES, WIDE>(h, (const TH*)d.h + row * d.ldh, lane, d.d, on);
      gn_load<TX, NE, V, LANES, WIDE>(x, (const TX*)d.x + row * d.ldx, lane, d.d, on && d.pre);
      gn_load<TH, NE, V, LANES, WIDE>(dy, (const TH*)d.dy + row * d.lddy, lane, d.d, on && d.pre);
      gn_load<TX, NE, V, LANES, WIDE>(t, (const TX*)d.dx1 + row * d.lddx1, lane, d.d, on && d.dx1);
      if constexpr (PER_ROW) gn_load<float, NE, V, LANES, WIDE>(gr, d.gate + row * d.d, lane, d.d, on);
      if (d.post) {
#pragma unroll
        for (int i = 0; i < N; i++) h[i] = gn_in<NE, V, LANES>(i, lane, d.d) ? (h[i] - st[0]) * st[1] : 0.f;   // hhat
      }
      if (d.pre) {
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < N; i++) {
          float n = __builtin_fmaf(h[i], gw[i], gb[i]);
          if constexpr (PER_ROW) n *= gr[i];
          x[i] = gn_in<NE, V, LANES>(i, lane, d.d) ? (__builtin_fmaf(d.res_scale, x[i], n) - st[2]) * st[3] : 0.f;   // xhat
          sw[i] += dy[i] * x[i];
          sb[i] += dy[i];
          dy[i] *= pw[i];
          s[0] += dy[i] * x[i];
          s[1] += dy[i];
        }
        red(s);
        const float m1 = s[0] / d.d, m0 = d.pre == 2 ? s[1] / d.d : 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) t[i] += gn_in<NE, V, LANES>(i, lane, d.d) ? (dy[i] - m0 - x[i] * m1) * st[3] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < N; i++) x[i] = t[i] * d.res_scale;   // dx
      if (on) gn_store<TX, NE, V, LANES, WIDE>(x, (TX*)d.dx + row * d.lddx, lane, d.d);
      if constexpr (PER_ROW) {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = t[i] * __builtin_fmaf(h[i], gw[i], gb[i]);   // this row's dgate
        if (on) gn_store<float, NE, V, LANES, WIDE>(x, d.dgate + row * d.d, lane, d.d);
#pragma unroll
        for (int i = 0; i < N; i++) t[i] *= gr[i];
      }
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < N; i++) {
        sa[i] += t[i] * h[i];
        sc[i] += t[i];
        t[i] *= gw[i];
        s[0] += t[i] * h[i];
        s[1] += t[i];
      }
      if (d.post) {
        red(s);
        const float m1 = s[0] / d.d, m0 = d.post == 2 ? s[1] / d.d : 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) t[i] = (t[i] - m0 - h[i] * m1) * st[1];
      }
      if (on) gn_store<TH, NE, V, LANES, WIDE>(t, (TH*)d.dh + row * d.lddh, lane, d.d);
    }
    float w[N], qw[N], qb[N];
    gn_param<NE, V, LANES, WIDE>(w, gated ? d.gate + g * d.d : nullptr, 1.f, lane, d.d);
#pragma unroll
    for (int i = 0; i < N; i++) { qw[i] = fold[i * 64 * WAVES + tid] + w[i] * sa[i]; qb[i] = fold[(N + i) * 64 * WAVES + tid] + w[i] * sc[i]; }
    if (gated) {
      gn_param<NE, V, LANES, WIDE>(w, d.post_w, 1.f, lane, d.d);
      gn_param<NE, V, LANES, WIDE>(gb, d.post_b, 0.f, lane, d.d);
#pragma unroll
      for (int i = 0; i < N; i++) sa[i] = w[i] * sa[i] + gb[i] * sc[i];
      flush(sa, s0 == g * rpg && s1 == (g + 1) * rpg ? d.dgate + g * d.d : part.base + ((long long)4 * part.C + 2 * blockIdx.x + (s0 == c0 ? 0 : 1)) * d.d);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < N; i++) { fold[i * 64 * WAVES + tid] = qw[i]; fold[(N + i) * 64 * WAVES + tid] = qb[i]; }   // (read again by the same thread)
    s0 = s1;
  }
  float qw[N], qb[N];
#pragma unroll
  for (int i = 0; i < N; i++) { qw[i] = fold[i * 64 * WAVES + tid]; qb[i] = fold[(N + i) * 64 * WAVES + tid]; }
  if (d.dpre_w) flush(sw, part.base + (long long)blockIdx.x * d.d);
  if (d.dpre_b) flush(sb, part.base + ((long long)part.C + blockIdx.x) * d.d);
  if (d.dpost_w) flush(qw, part.base + ((long long)2 * part.C + blockIdx.x) * d.d);
  if (d.dpost_b) flush(qb, part.base + ((long long)3 * part.C + blockIdx.x) * d.d);
}

// sums of the workgroups, in their order: blockIdx.y 0..3 the four parameter vectors, the others the gate rows; 64 columns a block, 16 waves share the workgroups
__global__ __launch_bounds__(1024) void gated_norm_finish_kernel(GatedNormDesc d, GnPart part, long long gates) {
  __shared__ float fold[16][64];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, col = blockIdx.x * 64 + l;
  // rows `step` apart of the workgroups [lo, hi), the first one's `first` further on
  auto sum = [&](const float* from, int step, int first, long long lo, long long hi, float* out) {
    float s = 0.f;
    if (col < d.d) {
#pragma unroll 8
      for (long long i = lo + w; i < hi; i += 16) s += from[(i * step + (i == lo ? first : 0)) * d.d + col];
    }
    fold[w][l] = s;
    __syncthreads();
    if (w == 0 && col < d.d) {
      s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) s += fold[i][l];
      out[col] = s;
    }
    __syncthreads();
  };
  if (blockIdx.y < 4) {
    float* out = blockIdx.y == 0 ? d.dpre_w : blockIdx.y == 1 ? d.dpre_b : blockIdx.y == 2 ? d.dpost_w : d.dpost_b;
    if (out) sum(part.base + (long long)blockIdx.y * part.C * d.d, 1, 0, 0, part.C, out);
    return;
  }
  for (long long g = blockIdx.y - 4; g < gates; g += gridDim.y - 4) {
    const long long r0 = g * d.rows_per_gate, r1 = r0 + d.rows_per_gate, lo = r0 / part.chunk, hi = (r1 - 1) / part.chunk + 1;
    // (one workgroup that held all of a gate's rows has written the sum itself)
    if (hi - lo > 1) sum(part.base + (long long)4 * part.C * d.d, 2, r0 == lo * part.chunk ? 0 : 1, lo, hi, d.dgate + g * d.d);
  }
}

// waves a row
static int gn_waves(int d) { return d <= 768 ? 1 : d <= 1024 ? 2 : d <= 2048 ? 4 : d <= 4096 ? 8 : 16; }
static GnPart gn_part(const GatedNormDesc& d, void* ws) {
  // the workgroups that the chip holds at once (waves a SIMD as the kernel's comment has them: 1024 runs of rows where 768 fit, 7108 x 1001: 41 us instead of 32);
  // a run of rows is a whole number of the teams' rounds
  const int k = gn_waves(d.d), teams = k > 4 ? 1 : 4 / k, wgs = k > 4 ? 4096 / k : (d.d > 512 && d.d <= 768) || (d.d & 7) ? 768 : 1024;
  GnPart p;
  p.chunk = (((d.rows + wgs - 1) / wgs + teams - 1) / teams) * teams;
  p.C = (int)((d.rows + p.chunk - 1) / p.chunk);
  p.base = (float*)ws;
  return p;
}
static long long gn_gates(const GatedNormDesc& d) { return d.gate && d.rows_per_gate > 1 ? d.rows / d.rows_per_gate : 0; }

size_t gated_norm_bwd_workspace_bytes(const GatedNormDesc& d) {
  if (d.rows <= 0 || d.d <= 0) return 256;
  const GnPart p = gn_part(d, nullptr);
  return (size_t)(gn_gates(d) ? 6 : 4) * p.C * d.d * sizeof(float) + 256;
}

static int gn_check(const GatedNormDesc& d, int ht, int xt, bool bwd, const char* what, bool& wide) {
  if (d.rows < 0 || d.rows >= (1ll << 31) || d.d <= 0 || d.d > 8192) { set_error("%s: %lld rows of %d (rows up to 8192 wide)", what, d.rows, d.d); return SMBV_ERR_SHAPE; }
  if (ht < 0 || ht > 2 || xt < 0 || xt > 2 || (xt != ht && xt != 2)) { set_error("%s: the residual stream has the block's type or fp32", what); return SMBV_ERR_ARG; }
  if (d.post < 0 || d.post > 2 || d.pre < 0 || d.pre > 2) { set_error("%s: unknown norm", what); return SMBV_ERR_ARG; }
  if ((!d.post && (d.post_w || d.post_b)) || (!d.pre && (d.pre_w || d.pre_b))) { set_error("%s: a weight or bias without its norm", what); return SMBV_ERR_ARG; }
  if (d.gate && (d.rows_per_gate <= 0 || d.rows % d.rows_per_gate)) { set_error("%s: %lld rows are not whole groups of %lld", what, d.rows, d.rows_per_gate); return SMBV_ERR_SHAPE; }
  if (!(d.eps >= 0.f)) { set_error("%s: eps must not be negative", what); return SMBV_ERR_ARG; }
  if (d.rows == 0) return SMBV_OK;
  if (!d.h || !d.x || !d.stats || (!bwd && (!d.x1 || (d.pre && !d.y)))) { set_error("%s: null operand", what); return SMBV_ERR_ARG; }
  if (bwd && (!d.dh || !d.dx || (d.pre && !d.dy) || (!d.pre && !d.dx1) || (d.gate && !d.dgate))) { set_error("%s: null operand", what); return SMBV_ERR_ARG; }
  if (bwd && ((d.dpost_w && !d.post_w) || (d.dpost_b && !d.post_b) || (d.dpre_w && !d.pre_w) || (d.dpre_b && !d.pre_b) || (d.dgate && !d.gate))) { set_error("%s: the gradient of an absent parameter", what); return SMBV_ERR_ARG; }
  const long long lds[] = {d.ldh, d.ldx, d.ldx1, d.ldy, d.lddx1, d.lddy, d.lddh, d.lddx};
  const void* ps[] = {d.h, d.x, d.x1, d.y, d.dx1, d.dy, d.dh, d.dx};
  const int types[] = {ht, xt, xt, ht, xt, ht, ht, xt};
  long long bits = d.d;
  uintptr_t addr = 0;
  for (int i = 0; i < 8; i++) {
    if (!ps[i]) continue;
    if ((uintptr_t)ps[i] & (types[i] == 2 ? 3 : 1)) { set_error("%s: alignment", what); return SMBV_ERR_ALIGN; }
    if (lds[i] < d.d) { set_error("%s: a row stride of %lld for rows of %d", what, lds[i], d.d); return SMBV_ERR_SHAPE; }
    bits |= lds[i];
    addr |= (uintptr_t)ps[i];
  }
  const void* fs[] = {d.post_w, d.post_b, d.gate, d.pre_w, d.pre_b, d.dgate, d.dpost_w, d.dpost_b, d.dpre_w, d.dpre_b};
  for (const void* p : fs) {
    if ((uintptr_t)p & 3) { set_error("%s: alignment", what); return SMBV_ERR_ALIGN; }
    addr |= (uintptr_t)p;
  }
  if ((uintptr_t)d.stats & 15) { set_error("%s: stats must be 16-byte aligned", what); return SMBV_ERR_ALIGN; }
  wide = (bits & 7) == 0 && (addr & 15) == 0;
  return SMBV_OK;
}

// elements and their vectors a lane, waves a row
#define GN_SHAPES(GO)                                                                     \
  if (d.d <= 512) GO(8, 8, 1)                                                             \
  else if (d.d <= 768) GO(12, 4, 1)                                                       \
  else if (d.d <= 1024) GO(8, 8, 2)                                                       \
  else if (d.d <= 2048) GO(8, 8, 4)                                                       \
  else if (d.d <= 4096) GO(8, 8, 8)                                                       \
  else GO(8, 8, 16)

template <class TH, class TX>
static void gn_fwd(const GatedNormDesc& d, bool wide, hipStream_t st) {
  const int k = gn_waves(d.d), teams = k > 4 ? 1 : 4 / k;
  const dim3 grid((unsigned)std::min<long long>((d.rows + teams - 1) / teams, 2048)), blk(k > 4 ? 64 * k : 256);   // eight workgroups a CU walk the rows
#define GO(NE, V, K) { if (wide) hipLaunchKernelGGL((gated_norm_fwd_kernel<TH, TX, NE, V, K, true>), grid, blk, 0, st, d); \
                       else hipLaunchKernelGGL((gated_norm_fwd_kernel<TH, TX, NE, V, K, false>), grid, blk, 0, st, d); }
  GN_SHAPES(GO)
#undef GO
}
template <class TH, class TX>
static void gn_bwd(const GatedNormDesc& d, bool wide, const GnPart& part, hipStream_t st) {
  const int k = gn_waves(d.d);
  const dim3 grid(part.C), blk(k > 4 ? 64 * k : 256);
  const bool per_row = d.gate && d.rows_per_gate == 1;
#define GO1(NE, V, K, W) { if (per_row) hipLaunchKernelGGL((gated_norm_bwd_kernel<TH, TX, NE, V, K, W, true>), grid, blk, 0, st, d, part); \
                           else hipLaunchKernelGGL((gated_norm_bwd_kernel<TH, TX, NE, V, K, W, false>), grid, blk, 0, st, d, part); }
#define GO(NE, V, K) { if (wide) GO1(NE, V, K, true) else GO1(NE, V, K, false) }
  GN_SHAPES(GO)
#undef GO
}
#define GN_TYPES(FN, ...)                                                       \
  if (ht == 0) { if (xt == 0) FN<__bf16, __bf16>(__VA_ARGS__); else FN<__bf16, float>(__VA_ARGS__); }            \
  else if (ht == 1) { if (xt == 1) FN<_Float16, _Float16>(__VA_ARGS__); else FN<_Float16, float>(__VA_ARGS__); } \
  else FN<float, float>(__VA_ARGS__);

int gated_norm_fwd(const GatedNormDesc& d, int ht, int xt, hipStream_t st) {
  bool wide = false;
  if (int rc = gn_check(d, ht, xt, false, "gated_norm_fwd", wide)) return rc;
  if (d.rows == 0) return SMBV_OK;
  GN_TYPES(gn_fwd, d, wide, st)
  return check_launch("gated_norm_fwd");
}

int gated_norm_bwd(const GatedNormDesc& d, int ht, int xt, void* ws, size_t ws_bytes, hipStream_t st) {
  bool wide = false;
  if (int rc = gn_check(d, ht, xt, true, "gated_norm_bwd", wide)) return rc;
  if (d.rows == 0) return SMBV_OK;
  const size_t need = gated_norm_bwd_workspace_bytes(d);
  if (!ws || ws_bytes < need || ((uintptr_t)ws & 255)) { set_error("gated_norm_bwd: workspace short or not 256-byte aligned (%zu < %zu)", ws_bytes, need); return SMBV_ERR_WORKSPACE; }
  const GnPart part = gn_part(d, ws);
  GN_TYPES(gn_bwd, d, wide, part, st)
  const long long gates = gn_gates(d);
  hipLaunchKernelGGL(gated_norm_finish_kernel, dim3((d.d + 63) / 64, 4 + (unsigned)std::min<long long>(gates, 512)), dim3(1024), 0, st, d, part, gates);
  return check_launch("gated_norm_bwd");
}

}  // namespace smbv
