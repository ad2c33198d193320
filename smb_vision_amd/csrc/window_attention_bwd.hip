// Windowed attention with sinks, backward (window_attention.h has the definition).  With P from the stored LSE and delta_i = sum_d dO_id O_id:
//     dS_ij = P_ij (dO_i V_j - delta_i),   dQ_i = scale sum_j dS_ij K_j,   dK_j = scale sum_i dS_ij Q_i,   dV_j = sum_i P_ij dO_i
// as three launches without atomics, so that a repeated call gives the same bits:
//   delta     one wave a row
//   dQ        128 rows a workgroup, walking their keys (the forward's loop): S^T and dP^T by one product each, dQ^T += K^T dS^T
//   dK, dV    128 keys a workgroup (32 a wave, K and V in registers), walking the rows that see them - all G heads of the group, which is where the sum over
//             a shared key head's queries is formed: S and dP by one product each, dV^T += dO^T P, dK^T += Q^T dS
// S and dP are formed twice (7 products instead of 5): the alternative is dQ by float atomics, whose order changes the result.
// P and dS are rounded to 16 bits for the second products, which add in 32 bits.  fp16 has a narrow exponent: gradients of 2^-20 would be lost in dS.  So dS is
// formed in units of a power of two: dQ's workgroup takes dO times 2^-e, e the exponent of the row's largest |dO| (exact), dK's keeps its accumulator in
// units of 2^e, e the largest exponent among the rows met so far, and rescales it when that grows.
#include "window_attention.h"
#include <math.h>

namespace smbv {

// fp16: exponent of a row's largest |dO| (0 for a row of zeros or with an infinity), beside delta in the workspace
static constexpr int WIN_NO_EXP = -1000;

template <class E>
__global__ __launch_bounds__(256) void win_delta_kernel(WinDesc d, int* __restrict__ expo) {
  const int l = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), n = (long long)d.B * d.H * d.Sq;   // [b][i][h], heads fastest
  if (row >= n) return;
  const int h = (int)(row % d.H);
  const long long bi = row / d.H;
  const int i = (int)(bi % d.Sq), b = (int)(bi / d.Sq);
  const WinSeq seq = win_seq(d, b);
  float s = 0.f, mx = 0.f;
  if (i < seq.qlen && 2 * l < d.D) {
    const unsigned g = *(const unsigned*)(d.g + b * d.sg.b + i * d.sg.r + h * d.sg.h + 2 * l);
    const long long oo = b * d.so.b + i * d.so.r + h * d.so.h + 2 * l;
    const unsigned o = *(const unsigned*)(d.o_in + oo), lo = d.o_lo_in ? *(const unsigned*)(d.o_lo_in + oo) : 0u;
    const float g0 = el_f<E>((uint16_t)g), g1 = el_f<E>((uint16_t)(g >> 16));
    s = g0 * (el_f<E>((uint16_t)o) + el_f<E>((uint16_t)lo)) + g1 * (el_f<E>((uint16_t)(o >> 16)) + el_f<E>((uint16_t)(lo >> 16)));
    mx = fmaxf(fabsf(g0), fabsf(g1));
  }
  s = wave_sum(s);
  const long long out = ((long long)b * d.H + h) * d.Sq + i;
  if (l == 0) d.delta[out] = s;
  if constexpr (E::half) {
    mx = wave_max(mx);
    if (l == 0) expo[out] = mx > 0.f && mx < INFINITY ? ilogbf(mx) : WIN_NO_EXP;
  }
}

template <class E, int DP>
__global__ __launch_bounds__(256, DP == 128 ? 2 : 3) void win_dq_kernel(WinDesc d, const int* __restrict__ expo) {
  constexpr int KS = DP / 16, DT = DP / 32, IMG = 64 * DP * 2;
  using v8 = typename E::v8;
  __shared__ __attribute__((aligned(16))) unsigned char smem[4 * IMG];   // two slots of K | V
  const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), r31 = l & 31, h2 = l >> 5;
  int tile, hk, b;
  xcd_block_order((int)(((long long)d.Sq * d.G + 127) / 128), d.Hk, tile, hk, b);
  const WinSeq seq = win_seq(d, b);
  const int r0 = tile * 128, rows = d.Sq * d.G;
  const int i0 = win_div(d, r0), i1 = min(seq.qlen, win_div(d, min(r0 + 127, rows - 1)) + 1);
  const WinKeys wk = win_keys(d, seq, i0, i1);
  const int r = r0 + 32 * w + r31, i = win_div(d, r), head = hk * d.G + (r - i * d.G);
  const bool live = r < rows && i < seq.qlen;
  WinRow wr = win_row(d, seq, i);
  if (!live) wr.hi = -1;
  const uint16_t* kb = d.k + b * d.sk.b + hk * d.sk.h;
  const uint16_t* vb = d.v + b * d.sv.b + hk * d.sv.h;
  const float c = d.scale * 1.4426950408889634f;
  float lse2 = INFINITY, delta = 0.f;
  int e = 0;
  if (live) {
    const long long at = ((long long)b * d.H + head) * d.Sq + i;
    const float ls = d.lse[at];
    if (ls != -INFINITY) lse2 = ls * 1.4426950408889634f;   // (an empty row: exp2(s - inf) = 0)
    delta = d.delta[at];
    if constexpr (E::half) {
      e = expo[at];
      if (e == WIN_NO_EXP) e = 0;
      delta = ldexpf(delta, -e);
    }
  }
  v8 qf[KS], gf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    const int ch = 16 * ks + 8 * h2;
    if (live && ch < d.D) {
      x = *(const u32x4*)(d.q + b * d.sq.b + i * d.sq.r + head * d.sq.h + ch);
      y = *(const u32x4*)(d.g + b * d.sg.b + i * d.sg.r + head * d.sg.h + ch);
    }
    qf[ks] = __builtin_bit_cast(v8, x);
    gf[ks] = __builtin_bit_cast(v8, y);
    if constexpr (E::half) {
#pragma unroll
      for (int k = 0; k < 8; k++) gf[ks][k] = (_Float16)ldexpf((float)gf[ks][k], -e);
    }
  }
  f32x16 acc[DT], cdel;   // cdel: -delta, the start of every dP product
#pragma unroll
  for (int x = 0; x < 16; x++) {
#pragma unroll
    for (int dt = 0; dt < DT; dt++) acc[dt][x] = 0.f;
    cdel[x] = -delta;
  }
  const int nt = (wk.n + 63) / 64;
  const int wi0 = win_div(d, r0 + 32 * w), wi1 = min(seq.qlen, win_div(d, min(r0 + 32 * w + 31, rows - 1)) + 1);   // this wave's queries
  const WinCopy<DP> copy(w, l, d.D);
  unsigned koff[WinCopy<DP>::NP], voff[WinCopy<DP>::NP];
  copy.offsets(koff, d.sk.r);
  copy.offsets(voff, d.sv.r);
  const unsigned lds = __builtin_amdgcn_readfirstlane((int)(lds_addr_of(smem) + w * (IMG / 4)));
  auto stage = [&](int j, int slot) __attribute__((always_inline)) {
    copy.keys(kb, d.sk.r, koff, wk, 64 * j, lds + slot * 2 * IMG);
    copy.keys(vb, d.sv.r, voff, wk, 64 * j, lds + slot * 2 * IMG + IMG);
  };
  auto keys = [&](int j, const unsigned char* img) __attribute__((always_inline)) {
    const int kind = win_tile(d, seq, wk, 64 * j, wi0, wi1);
    if (kind == 0) return;
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
      f32x16 s, dp;
#pragma unroll
      for (int x = 0; x < 16; x++) s[x] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        s = E::mfma(__builtin_bit_cast(v8, *(const u32x4*)(img + win_img<DP>(32 * kt + r31, 2 * ks + h2))), qf[ks], s);
        dp = E::mfma(__builtin_bit_cast(v8, *(const u32x4*)(img + IMG + win_img<DP>(32 * kt + r31, 2 * ks + h2))), gf[ks], ks == 0 ? cdel : dp);
      }
      if (kind == 1) {
#pragma unroll
        for (int x = 0; x < 16; x++) {
          const int u = 64 * j + 32 * kt + win_acc_row(x, l), key = u < wk.ns ? u : u + wk.jump;
          const bool vis = u < wk.n && key <= wr.hi && (key >= wr.lo || key < d.sinks);
          s[x] = vis ? s[x] : -INFINITY;
          dp[x] = vis ? dp[x] : 0.f;
        }
      }
#pragma unroll
      for (int half = 0; half < 2; half++) {
        v8 ds;
#pragma unroll
        for (int x = 0; x < 8; x++) ds[x] = (typename E::e)(fast_exp2(__builtin_fmaf(s[8 * half + x], c, -lse2)) * dp[8 * half + x]);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) acc[dt] = E::mfma(__builtin_bit_cast(v8, win_read_tr<DP>(img, 32 * kt + 16 * half, dt, l)), ds, acc[dt]);
      }
    }
  };
  if (nt > 0) stage(0, 0);
  for (int j = 0; j < nt; j += 2) {
    win_arrived();
    if (j + 1 < nt) stage(j + 1, 1);
    keys(j, smem);
    if (j + 1 >= nt) break;
    win_arrived();
    if (j + 2 < nt) stage(j + 2, 0);
    keys(j + 1, smem + 2 * IMG);
  }
  if (r >= rows) return;
  uint16_t* out = d.dq + b * d.sdq.b + i * d.sdq.r + head * d.sdq.h;
  const float f = E::half ? ldexpf(d.scale, e) : d.scale;
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int rg = 0; rg < 4; rg++) {
      const int d0 = 32 * dt + 8 * rg + 4 * h2;
      if (d0 < d.D)
        *(u32x2*)(out + d0) = (u32x2){el_pack<E>(acc[dt][4 * rg] * f, acc[dt][4 * rg + 1] * f), el_pack<E>(acc[dt][4 * rg + 2] * f, acc[dt][4 * rg + 3] * f)};
    }
}

// rows [lo, hi) (r = i G + g) that see any of the keys [k0, k1)
__device__ __forceinline__ void win_key_rows(const WinDesc& d, const WinSeq& s, int k0, int k1, int& lo, int& hi) {
  k1 = min(k1, s.klen);
  int ilo = d.right < 0 ? 0 : max(0, k0 - d.right - s.shift);
  int ihi = d.left < 0 || k0 < d.sinks ? s.qlen : min(s.qlen, k1 - 1 + d.left - s.shift + 1);
  if (k0 >= k1 || ihi <= ilo) ilo = ihi = 0;
  lo = ilo * d.G;
  hi = ihi * d.G;
}

// rows q0 .. q0 + 63 of a key head's queries and their gradients (rows past rhi take row rhi - 1: their LSE is set to +inf).  A tile starts at a whole query
// when 64 is a multiple of G, and its rows then lie at fixed distances.
template <int DP>
__device__ __forceinline__ void win_copy_rows(const WinCopy<DP>& c, const WinDesc& d, const uint16_t* base, const WinStride& st, const unsigned (&off)[WinCopy<DP>::NP],
                                              int q0, int rhi, bool fixed, unsigned lds) {
  if (fixed && q0 + 64 <= rhi) {
    const uint16_t* s = win_uniform(base + (long long)win_div(d, q0) * st.r);
#pragma unroll
    for (int p = 0; p < WinCopy<DP>::NP; p++) win_dma_off(s, off[p], lds + p * 1024);
  } else {
#pragma unroll
    for (int p = 0; p < WinCopy<DP>::NP; p++) {
      const int r = min(q0 + c.row[p], rhi - 1), i = win_div(d, r);
      win_dma_ptr(base + (long long)i * st.r + (long long)(r - i * d.G) * st.h + c.chunk[p] * 8, lds + p * 1024);
    }
  }
}

struct WinRowStat { float lse, delta; int expo; };

// How the rows that see a tile of 128 keys are shared out.  The first `nsink` tiles hold sinks, which EVERY later row sees: alone they would run as long as all
// rows are, 320 tiles of rows against 66 at 20,480 tokens and a window of 4097.  So their rows go to c1 workgroups, the other tiles' to c2 (1 unless there are too
// few tiles to fill the chip); a tile's workgroups leave their fp32 sums in the workspace and a second launch adds them in order.
struct WinSplit {
  int tiles, nsink, c1, c2, units;  // units: workgroups of one key head
  float* part;                      // [B, Hk][slots][dK | dV][128 keys][DP]
};
__device__ __forceinline__ int win_split_slots(const WinSplit& s) { return (s.c1 > 1 ? s.nsink * s.c1 : 0) + (s.c2 > 1 ? (s.tiles - s.nsink) * s.c2 : 0); }

template <class E, int DP>
__global__ __launch_bounds__(256, 2) void win_dkv_kernel(WinDesc d, const int* __restrict__ expo, WinSplit sp) {
  constexpr int KS = DP / 16, DT = DP / 32, IMG = 64 * DP * 2;
  using v8 = typename E::v8;
  constexpr int STAT = 64 * 5 * 4;   // LSE | delta | lo | hi | exponent of a tile's rows
  __shared__ __attribute__((aligned(16))) unsigned char smem[4 * IMG + 2 * STAT];   // two slots of Q | dO, two of the rows' numbers
  const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), r31 = l & 31, h2 = l >> 5;
  int unit, hk, b;
  xcd_block_order(sp.units, d.Hk, unit, hk, b);
  const bool sink = unit < sp.nsink * sp.c1;
  const int c12 = sink ? sp.c1 : sp.c2, rest = sink ? unit : unit - sp.nsink * sp.c1, tile = (sink ? 0 : sp.nsink) + rest / c12, share = rest % c12;
  const WinSeq seq = win_seq(d, b);
  const int k0 = tile * 128, kw0 = k0 + 32 * w, key = kw0 + r31;
  int rlo, rhi;
  win_key_rows(d, seq, k0, k0 + 128, rlo, rhi);
  if (c12 > 1) {   // whole tiles of 64 rows to a share
    const long long n = (rhi - rlo + 63) / 64;
    const int lo = rlo + (int)(n * share / c12) * 64;
    rhi = min(rhi, rlo + (int)(n * (share + 1) / c12) * 64);
    rlo = lo;
  }
  const float c = d.scale * 1.4426950408889634f;
  v8 kf[KS], vf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    const int ch = 16 * ks + 8 * h2;
    if (key < seq.klen && ch < d.D) {
      x = *(const u32x4*)(d.k + b * d.sk.b + key * d.sk.r + hk * d.sk.h + ch);
      y = *(const u32x4*)(d.v + b * d.sv.b + key * d.sv.r + hk * d.sv.h + ch);
    }
    kf[ks] = __builtin_bit_cast(v8, x);
    vf[ks] = __builtin_bit_cast(v8, y);
  }
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int x = 0; x < 16; x++) { dk[dt][x] = 0.f; dv[dt][x] = 0.f; }
  int emax = WIN_NO_EXP;
  const WinCopy<DP> copy(w, l, d.D);
  unsigned qoff[WinCopy<DP>::NP], goff[WinCopy<DP>::NP];
#pragma unroll
  for (int p = 0; p < WinCopy<DP>::NP; p++) {
    const int i = win_div(d, copy.row[p]), g = copy.row[p] - i * d.G;
    qoff[p] = (unsigned)(i * (unsigned)d.sq.r + g * (unsigned)d.sq.h) * 2 + copy.chunk[p] * 16;
    goff[p] = (unsigned)(i * (unsigned)d.sg.r + g * (unsigned)d.sg.h) * 2 + copy.chunk[p] * 16;
  }
  const bool fixed = 64 % d.G == 0;
  const uint16_t* qb = d.q + b * d.sq.b + (long long)hk * d.G * d.sq.h;
  const uint16_t* gb = d.g + b * d.sg.b + (long long)hk * d.G * d.sg.h;
  const unsigned lds = __builtin_amdgcn_readfirstlane((int)(lds_addr_of(smem) + w * (IMG / 4)));
  auto stage = [&](int q0, int slot) __attribute__((always_inline)) {
    win_copy_rows<DP>(copy, d, qb, d.sq, qoff, q0, rhi, fixed, lds + slot * 2 * IMG);
    win_copy_rows<DP>(copy, d, gb, d.sg, goff, q0, rhi, fixed, lds + slot * 2 * IMG + IMG);
  };
  // the first wave's lanes fetch a row's numbers a tile ahead and put them into LDS behind the products
  auto fetch = [&](int q0) __attribute__((always_inline)) {
    WinRowStat x = {INFINITY, 0.f, WIN_NO_EXP};
    const int r = q0 + t;
    if (t < 64 && r < rhi) {
      const int i = win_div(d, r);
      const long long at = ((long long)b * d.H + hk * d.G + (r - i * d.G)) * d.Sq + i;
      const float ls = d.lse[at];
      x.lse = ls == -INFINITY ? INFINITY : ls * 1.4426950408889634f;
      x.delta = d.delta[at];
      if constexpr (E::half) x.expo = expo[at];
    }
    return x;
  };
  auto put = [&](const WinRowStat& x, int q0, int slot) __attribute__((always_inline)) {
    if (t < 64) {
      unsigned char* at = smem + 4 * IMG + slot * STAT + 4 * t;
      const WinRow wr = win_row(d, seq, win_div(d, q0 + t));
      *(float*)at = x.lse;
      *(float*)(at + 256) = -x.delta;
      *(int*)(at + 512) = wr.lo;
      *(int*)(at + 768) = q0 + t < rhi ? wr.hi : -1;
      if constexpr (E::half) *(int*)(at + 1024) = x.expo;
    }
  };
  auto rowtile = [&](int q0, const unsigned char* img, const unsigned char* st) __attribute__((always_inline)) {
    const int pa = win_div(d, q0) + seq.shift, pb = win_div(d, min(q0 + 64, rhi) - 1) + seq.shift, klast = min(kw0 + 32, seq.klen) - 1;
    if (kw0 > klast || (d.right >= 0 && kw0 > pb + d.right) || (d.left >= 0 && kw0 >= d.sinks && klast < pa - d.left)) return;   // nobody sees these keys
    const bool all = (d.right < 0 || klast <= pa + d.right) && (d.left < 0 || klast < d.sinks || kw0 >= pb - d.left);
    float unit = 1.f;
    if constexpr (E::half) {
      int e = *(const int*)(st + 1024 + 4 * l);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) e = max(e, __shfl_xor(e, o, 64));
      if (e > emax) {
        const float f = emax == WIN_NO_EXP ? 0.f : ldexpf(1.f, emax - e);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int x = 0; x < 16; x++) dk[dt][x] *= f;
        emax = e;
      }
      unit = emax == WIN_NO_EXP ? 1.f : ldexpf(1.f, -emax);
    }
#pragma unroll
    for (int qt = 0; qt < 2; qt++) {
      f32x16 s, dp;
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const f32x4 de = *(const f32x4*)(st + 256 + (32 * qt + 8 * x + 4 * h2) * 4);
#pragma unroll
        for (int y = 0; y < 4; y++) { s[4 * x + y] = 0.f; dp[4 * x + y] = de[y]; }
      }
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        s = E::mfma(__builtin_bit_cast(v8, *(const u32x4*)(img + win_img<DP>(32 * qt + r31, 2 * ks + h2))), kf[ks], s);
        dp = E::mfma(__builtin_bit_cast(v8, *(const u32x4*)(img + IMG + win_img<DP>(32 * qt + r31, 2 * ks + h2))), vf[ks], dp);
      }
      if (!all) {
#pragma unroll
        for (int x = 0; x < 16; x++) {
          const int row = 32 * qt + win_acc_row(x, l);
          const bool vis = key <= *(const int*)(st + 768 + 4 * row) && (key >= *(const int*)(st + 512 + 4 * row) || key < d.sinks);
          s[x] = vis ? s[x] : -INFINITY;
          dp[x] = vis ? dp[x] : 0.f;
        }
      }
#pragma unroll
      for (int half = 0; half < 2; half++) {
        v8 pf, ds;
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const f32x4 ls = *(const f32x4*)(st + (32 * qt + 16 * half + 8 * x + 4 * h2) * 4);
#pragma unroll
          for (int y = 0; y < 4; y++) {
            const float p = fast_exp2(__builtin_fmaf(s[8 * half + 4 * x + y], c, -ls[y]));
            pf[4 * x + y] = (typename E::e)p;
            float g = p * dp[8 * half + 4 * x + y];
            if constexpr (E::half) g *= unit;
            ds[4 * x + y] = (typename E::e)g;
          }
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
          dv[dt] = E::mfma(__builtin_bit_cast(v8, win_read_tr<DP>(img + IMG, 32 * qt + 16 * half, dt, l)), pf, dv[dt]);
          dk[dt] = E::mfma(__builtin_bit_cast(v8, win_read_tr<DP>(img, 32 * qt + 16 * half, dt, l)), ds, dk[dt]);
        }
      }
    }
  };
  if (rlo < rhi) {
    stage(rlo, 0);
    put(fetch(rlo), rlo, 0);
  }
  for (int q0 = rlo; q0 < rhi; q0 += 128) {
    win_arrived();
    WinRowStat next = {INFINITY, 0.f, WIN_NO_EXP};
    if (q0 + 64 < rhi) { stage(q0 + 64, 1); next = fetch(q0 + 64); }
    rowtile(q0, smem, smem + 4 * IMG);
    if (q0 + 64 >= rhi) break;
    put(next, q0 + 64, 1);
    win_arrived();
    if (q0 + 128 < rhi) { stage(q0 + 128, 0); next = fetch(q0 + 128); }
    rowtile(q0 + 64, smem + 2 * IMG, smem + 4 * IMG + STAT);
    if (q0 + 128 < rhi) put(next, q0 + 128, 0);
  }
  const float f = E::half && emax != WIN_NO_EXP ? ldexpf(d.scale, emax) : d.scale;
  if (c12 > 1) {   // [32-channel block][key][32 channels]: a lane's four channels go out as 16 bytes
    const int slots = win_split_slots(sp), slot = sink || sp.c1 <= 1 ? rest : sp.nsink * sp.c1 + rest;
    float* part = sp.part + (((long long)b * d.Hk + hk) * slots + slot) * (2 * 128 * DP);
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int rg = 0; rg < 4; rg++) {
        float* at = part + (dt * 128 + 32 * w + r31) * 32 + 8 * rg + 4 * h2;
        *(f32x4*)at = (f32x4){dk[dt][4 * rg] * f, dk[dt][4 * rg + 1] * f, dk[dt][4 * rg + 2] * f, dk[dt][4 * rg + 3] * f};
        *(f32x4*)(at + 128 * DP) = (f32x4){dv[dt][4 * rg], dv[dt][4 * rg + 1], dv[dt][4 * rg + 2], dv[dt][4 * rg + 3]};
      }
    return;
  }
  if (key >= d.Sk) return;
  const bool live = key < seq.klen;
  uint16_t* ok = d.dk + b * d.sdk.b + key * d.sdk.r + hk * d.sdk.h;
  uint16_t* ov = d.dv + b * d.sdv.b + key * d.sdv.r + hk * d.sdv.h;
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int rg = 0; rg < 4; rg++) {
      const int d0 = 32 * dt + 8 * rg + 4 * h2;
      if (d0 >= d.D) continue;
      float a[4], e[4];
#pragma unroll
      for (int x = 0; x < 4; x++) { a[x] = live ? dk[dt][4 * rg + x] * f : 0.f; e[x] = live ? dv[dt][4 * rg + x] : 0.f; }
      *(u32x2*)(ok + d0) = (u32x2){el_pack<E>(a[0], a[1]), el_pack<E>(a[2], a[3])};
      *(u32x2*)(ov + d0) = (u32x2){el_pack<E>(e[0], e[1]), el_pack<E>(e[2], e[3])};
    }
}

// adds the shares of the tiles that were split: a workgroup 8 keys of one tile's dK or dV
template <class E, int DP>
__global__ __launch_bounds__(256) void win_dkv_join_kernel(WinDesc d, WinSplit sp) {
  constexpr int PER = DP / 4, KEYS = 256 / PER;   // four channels a thread
  const int split0 = sp.c1 > 1 ? 0 : sp.nsink, ntile = (sp.c2 > 1 ? sp.tiles : sp.nsink) - split0;   // the tiles [split0, split0 + ntile) were split
  const int groups = 128 / KEYS;
  long long x = blockIdx.x;
  const int part = (int)(x & 1);
  x >>= 1;
  const int kg = (int)(x % groups);
  x /= groups;
  const int tile = split0 + (int)(x % ntile);
  x /= ntile;
  const int hk = (int)(x % d.Hk), b = (int)(x / d.Hk);
  const bool sink = tile < sp.nsink;
  const int c12 = sink ? sp.c1 : sp.c2, slot0 = sink ? tile * sp.c1 : (sp.c1 > 1 ? sp.nsink * sp.c1 : 0) + (tile - sp.nsink) * sp.c2;
  const int kl = kg * KEYS + threadIdx.x / PER, ch = (threadIdx.x % PER) * 4, key = tile * 128 + kl;
  if (key >= d.Sk || ch >= d.D) return;
  const float* from = sp.part + (((long long)b * d.Hk + hk) * win_split_slots(sp) + slot0) * (2 * 128 * DP) + part * 128 * DP + ((ch >> 5) * 128 + kl) * 32 + (ch & 31);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < c12; i++) s += *(const f32x4*)(from + (long long)i * (2 * 128 * DP));
  if (key >= win_seq(d, b).klen) s = (f32x4){0.f, 0.f, 0.f, 0.f};
  const WinStride& st = part ? d.sdv : d.sdk;
  *(u32x2*)((part ? d.dv : d.dk) + b * st.b + key * st.r + hk * st.h + ch) = (u32x2){el_pack<E>(s[0], s[1]), el_pack<E>(s[2], s[3])};
}

static int win_dp(const WinDesc& d) { return d.D <= 32 ? 32 : d.D <= 64 ? 64 : 128; }
static WinSplit win_split(const WinDesc& d) {
  WinSplit s = {};
  s.tiles = (d.Sk + 127) / 128;
  s.nsink = d.left < 0 ? 0 : std::min(s.tiles, (int)(((long long)std::min(d.sinks, d.Sk) + 127) / 128));
  // rows that see a tile: all (a sink, an open window to the left), or those of a window
  const long long all = (long long)d.Sq * d.G, window = d.left < 0 || d.right < 0 ? all : std::min<long long>(all, ((long long)d.left + d.right + 128) * d.G);
  const long long plain = (long long)(s.tiles - s.nsink) * d.Hk * d.B;
  // A share costs its sums' way through memory (128 KiB at 128 channels, out and back) and saves a part of its tile's rows, a microsecond or two for 64 of them:
  // no share has less than 1024 rows, and the tiles are split only as far as there is room for more workgroups (two a CU; the sinks' four)
  s.c2 = (int)std::max<long long>(1, std::min<long long>({512 / std::max<long long>(plain, 1), window / 1024, 64}));
  const long long share = std::max<long long>(1024, (window + s.c2 - 1) / s.c2), sinks = (long long)s.nsink * d.Hk * d.B;
  s.c1 = (int)std::max<long long>(1, std::min<long long>({(all + share - 1) / share, 1024 / std::max<long long>(sinks, 1), 64}));
  if (s.nsink == s.tiles) s.c2 = 1;
  if (s.nsink == 0) s.c1 = 1;
  s.units = s.nsink * s.c1 + (s.tiles - s.nsink) * s.c2;
  return s;
}
static size_t win_split_bytes(const WinDesc& d, const WinSplit& s) {
  const size_t slots = (size_t)(s.c1 > 1 ? s.nsink * s.c1 : 0) + (size_t)(s.c2 > 1 ? (s.tiles - s.nsink) * s.c2 : 0);
  return slots * d.Hk * d.B * 2 * 128 * win_dp(d) * sizeof(float);
}

// workspace: delta fp32 [B, H, Sq] | exponents int32 [B, H, Sq] (fp16) | the shares of split key tiles
static size_t win_rows_bytes(const WinDesc& d) { return ((size_t)d.B * d.H * d.Sq * 4 + 255) & ~(size_t)255; }
size_t window_attention_bwd_workspace_bytes(const WinDesc& d, int dtype) {
  if (window_attention_check(d, true, "window_attention_bwd", true)) return 0;
  return win_rows_bytes(d) * (dtype ? 2 : 1) + win_split_bytes(d, win_split(d)) + 256;
}

template <class E>
static int win_bwd(WinDesc d, void* ws, hipStream_t st) {
  d.delta = (float*)ws;
  int* expo = (int*)((char*)ws + win_rows_bytes(d));
  const long long n = (long long)d.B * d.H * d.Sq;
  if (n > 0) {
    hipLaunchKernelGGL((win_delta_kernel<E>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, d, expo);
    const dim3 grid((unsigned)(((long long)d.Sq * d.G + 127) / 128 * d.Hk * d.B));
    if (d.D <= 32) hipLaunchKernelGGL((win_dq_kernel<E, 32>), grid, dim3(256), 0, st, d, expo);
    else if (d.D <= 64) hipLaunchKernelGGL((win_dq_kernel<E, 64>), grid, dim3(256), 0, st, d, expo);
    else hipLaunchKernelGGL((win_dq_kernel<E, 128>), grid, dim3(256), 0, st, d, expo);
  }
  if (d.Sk > 0) {
    WinSplit sp = win_split(d);
    sp.part = (float*)((char*)ws + win_rows_bytes(d) * (E::half ? 2 : 1));
    const dim3 grid((unsigned)((long long)sp.units * d.Hk * d.B));
    const int ntile = (sp.c1 > 1 ? sp.nsink : 0) + (sp.c2 > 1 ? sp.tiles - sp.nsink : 0);
#define GO(DP)                                                                                                                                    \
  {                                                                                                                                               \
    hipLaunchKernelGGL((win_dkv_kernel<E, DP>), grid, dim3(256), 0, st, d, expo, sp);                                                            \
    if (ntile) hipLaunchKernelGGL((win_dkv_join_kernel<E, DP>), dim3((unsigned)(2ll * (128 / (1024 / DP)) * ntile * d.Hk * d.B)), dim3(256), 0, st, d, sp); \
  }
    if (d.D <= 32) GO(32) else if (d.D <= 64) GO(64) else GO(128)
#undef GO
  }
  return check_launch("window_attention_bwd");
}

int window_attention_bwd(const WinDesc& d, int dtype, void* ws, size_t ws_bytes, hipStream_t st) {
  if (int rc = window_attention_check(d, true, "window_attention_bwd")) return rc;
  if (d.B == 0) return SMBV_OK;
  const size_t need = window_attention_bwd_workspace_bytes(d, dtype);
  if (!ws || ws_bytes < need || ((uintptr_t)ws & 255)) { set_error("window_attention_bwd: workspace short or not 256-byte aligned (%zu < %zu)", ws_bytes, need); return SMBV_ERR_WORKSPACE; }
  return dtype == 0 ? win_bwd<ElBf16>(d, ws, st) : win_bwd<ElF16>(d, ws, st);
}

}  // namespace smbv
