// Windowed attention with sinks, backward (window_attention.h has the definition).  With P from the stored LSE and delta_i = sum_d dO_id O_id:
//     dS_ij = P_ij (dO_i V_j - delta_i),   dQ_i = scale sum_j dS_ij K_j,   dK_j = scale sum_i dS_ij Q_i,   dV_j = sum_i P_ij dO_i
// in three launches without atomics, so that a repeated call gives the same bits:
//   rows      delta, and the row's LSE in log2 units, in the order in which the others walk the rows
//   dQ        32 rows a wave, walking their keys (the forward's loop): S^T and dP^T by one product each, dQ^T += K^T dS^T
//   dK, dV    32 keys a wave (K and V in registers), walking the rows that see them - all G heads of the group, which is where the sum over a shared key
//             head's queries is formed: S and dP by one product each, dV^T += dO^T P, dK^T += Q^T dS
// S and dP are formed twice (7 products instead of 5): the alternative is dQ by float atomics, whose order changes the result.
// P and dS are rounded to 16 bits for the second products, which add in 32 bits.  fp16 has a narrow exponent: gradients of 2^-20 would be lost in dS.  So dS is
// formed in units of a power of two: dQ's wave takes dO times 2^-e, e the exponent of the row's largest |dO| (exact), dK's keeps a key's accumulator in
// units of 2^e, e the largest exponent among the rows that the key has seen so far, and rescales it when that grows.  (Rows that it does not see do not count: one
// with a gradient 2^24 times the others' would take all their digits.)
#include "window_attention.h"
#include <limits.h>
#include <math.h>

namespace smbv {

// What the walks need of a row r = i G + g: [B, Hk][Sq G] each.  lse2: LSE in log2 units, +inf for a row that sees nothing (its exp2(s - lse2) is 0); ndelta: -delta;
// expo (fp16): exponent of the largest |dO|, WIN_NO_EXP for a row of zeros or with an infinity
struct WinRows { float *lse2, *ndelta; int* expo; };
static constexpr int WIN_NO_EXP = -1000;

// DP / 8 lanes a row, 16 bytes each (rows [b][i][h], heads fastest)
template <class E, int DP>
__global__ __launch_bounds__(256) void win_rows_kernel(WinDesc d, WinRows wr) {
  constexpr int L = DP / 8;
  const int c = (threadIdx.x % L) * 8;
  const long long row = (long long)blockIdx.x * (256 / L) + threadIdx.x / L, n = (long long)d.B * d.H * d.Sq;
  const bool on = row < n;
  const long long bi = on ? row / d.H : 0;
  const int h = on ? (int)(row - bi * d.H) : 0, b = (int)(bi / d.Sq), i = (int)(bi - (long long)b * d.Sq), hk = h / d.G, g = h - hk * d.G;
  const bool live = on && i < win_seq(d, b).qlen;
  float s = 0.f, mx = 0.f;
  if (live && c < d.D) {
    const long long oo = b * d.so.b + i * d.so.r + h * d.so.h + c;
    const u32x4 x = *(const u32x4*)(d.g + b * d.sg.b + i * d.sg.r + h * d.sg.h + c), o = *(const u32x4*)(d.o_in + oo);
    u32x4 lo = {0, 0, 0, 0};
    if (d.o_lo_in) lo = *(const u32x4*)(d.o_lo_in + oo);
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const int sh = 16 * (k & 1);
      const float gk = el_f<E>((uint16_t)(x[k >> 1] >> sh));
      s += gk * (el_f<E>((uint16_t)(o[k >> 1] >> sh)) + el_f<E>((uint16_t)(lo[k >> 1] >> sh)));
      mx = fmaxf(mx, fabsf(gk));
    }
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    if constexpr (E::half) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  }
  if (on && c == 0) {
    const long long at = (((long long)b * d.Hk + hk) * d.Sq + i) * d.G + g;
    const float ls = live ? d.lse[((long long)b * d.H + h) * d.Sq + i] : -INFINITY;
    wr.lse2[at] = ls == -INFINITY ? INFINITY : ls * 1.4426950408889634f;
    wr.ndelta[at] = ls == -INFINITY ? 0.f : -s;   // (a row that sees nothing gives no gradient, whatever its dO holds)
    if constexpr (E::half) wr.expo[at] = mx > 0.f && mx < INFINITY ? ilogbf(mx) : WIN_NO_EXP;
  }
}

template <class E, int DP, int NW, int NS, int OCC>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void win_dq_kernel(WinDesc d, WinRows wrows) {
  constexpr int KS = DP / 16, DT = DP / 32, IMG = 64 * DP * 2, BM = 32 * NW;
  using v8 = typename E::v8;
  using Copy = WinCopy<DP, NW>;
  __shared__ __attribute__((aligned(16))) unsigned char smem[NS * 2 * IMG];
  const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), r31 = l & 31, h2 = l >> 5;
  int tile, hk, b;
  win_block_order((int)(((long long)d.Sq * d.G + BM - 1) / BM), d.Hk, d.B, tile, hk, b);
  const WinSeq seq = win_seq(d, b);
  const int r0 = tile * BM, rows = d.Sq * d.G;
  const int i0 = win_div(d, r0), i1 = min(seq.qlen, win_div(d, min(r0 + BM, rows) - 1) + 1);
  const WinKeys wk = win_keys(d, seq, i0, i1);
  const int r = r0 + 32 * w + r31, i = win_div(d, r), head = hk * d.G + (r - i * d.G);
  const bool live = r < rows && i < seq.qlen;
  const WinView view = win_view(d, seq, wk, i);
  const uint16_t* kb = d.k + b * d.sk.b + hk * d.sk.h;
  const uint16_t* vb = d.v + b * d.sv.b + hk * d.sv.h;
  const float c = d.scale * 1.4426950408889634f;
  float lse2 = INFINITY, ndelta = 0.f;
  int e = 0;
  if (live) {
    const long long at = ((long long)b * d.Hk + hk) * rows + r;
    lse2 = wrows.lse2[at];
    ndelta = wrows.ndelta[at];
    if constexpr (E::half) {
      e = wrows.expo[at];
      if (e == WIN_NO_EXP) e = 0;
      ndelta = ldexpf(ndelta, -e);
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
    if (lse2 == INFINITY) { x = (u32x4){0, 0, 0, 0}; y = x; }   // the row sees nothing
    asm volatile("" : "+v"(x), "+v"(y));   // (waited for here, not in the loop)
    qf[ks] = __builtin_bit_cast(v8, x);
    gf[ks] = __builtin_bit_cast(v8, y);
    if constexpr (E::half) {
#pragma unroll
      for (int k = 0; k < 8; k++) gf[ks][k] = (_Float16)ldexpf((float)gf[ks][k], -e);
      asm volatile("" : "+v"(gf[ks]));
    }
  }
  f32x16 acc[DT], cdel;   // cdel: -delta, the start of every dP product
#pragma unroll
  for (int x = 0; x < 16; x++) {
#pragma unroll
    for (int dt = 0; dt < DT; dt++) acc[dt][x] = 0.f;
    cdel[x] = ndelta;
  }
  const int nt = (wk.n + 63) / 64;
  const int wi0 = win_div(d, r0 + 32 * w), wi1 = min(seq.qlen, win_div(d, min(r0 + 32 * w + 32, rows) - 1) + 1);   // this wave's queries
  const WinView v0 = win_view(d, seq, wk, wi0), v1 = win_view(d, seq, wk, wi1 - 1);
  const Copy copy(w, l, d.D);
  unsigned koff[Copy::NP], voff[Copy::NP];
  copy.offsets(koff, d.sk.r);
  copy.offsets(voff, d.sv.r);
  const unsigned lds = __builtin_amdgcn_readfirstlane((int)(lds_addr_of(smem) + w * (IMG / NW)));
  auto stage = [&](int j, int slot) __attribute__((always_inline)) {
    copy.keys(kb, d.sk.r, koff, wk, 64 * j, lds + slot * 2 * IMG);
    copy.keys(vb, d.sv.r, voff, wk, 64 * j, lds + slot * 2 * IMG + IMG);
  };
  WinRead<DP> rd(lds_addr_of(smem), l);
  auto keys = [&](int j, int off) __attribute__((always_inline)) {
    const int kind = wi0 < wi1 ? win_tile(v0, v1, 64 * j) : WIN_NONE;
    if (kind == WIN_NONE) return;
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
      f32x16 s, dp;
#pragma unroll
      for (int x = 0; x < 16; x++) s[x] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        s = E::mfma(__builtin_bit_cast(v8, rd.rows(ks, off + 64 * DP * kt)), qf[ks], s);
        dp = E::mfma(__builtin_bit_cast(v8, rd.rows(ks, off + IMG + 64 * DP * kt)), gf[ks], ks == 0 ? cdel : dp);
      }
      if (kind != WIN_ALL) win_mask(s, kind, view, 64 * j + 32 * kt + 4 * h2);   // (its exp2 is 0, and dP is finite as far as dO and V are)
#pragma unroll
      for (int half = 0; half < 2; half++) {
        v8 ds;
#pragma unroll
        for (int x = 0; x < 8; x++) ds[x] = (typename E::e)(fast_exp2(__builtin_fmaf(s[8 * half + x], c, -lse2)) * dp[8 * half + x]);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) acc[dt] = E::mfma(__builtin_bit_cast(v8, rd.cols(dt, off + 64 * DP * kt + 32 * DP * half)), ds, acc[dt]);
      }
    }
  };
  if (nt > 0) win_walk<NS, 2 * IMG>(nt, win_arrived<(NS - 2) * 2 * Copy::NP>, stage, keys, [&](int by) { rd.move(by); });
  if (r >= rows) return;
  uint16_t* out = d.dq + b * d.sdq.b + i * d.sdq.r + head * d.sdq.h;
  float f = d.scale;
  if (E::half && live) {   // (read again: a register less in the walk)
    e = wrows.expo[((long long)b * d.Hk + hk) * rows + r];
    if (e != WIN_NO_EXP) f = ldexpf(f, e);
  }
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int rg = 0; rg < 4; rg++) {
      const int d0 = 32 * dt + 8 * rg + 4 * h2;
      if (d0 >= d.D) continue;
      float a[4];
#pragma unroll
      for (int x = 0; x < 4; x++) a[x] = lse2 != INFINITY ? acc[dt][4 * rg + x] * f : 0.f;
      *(u32x2*)(out + d0) = (u32x2){el_pack<E>(a[0], a[1]), el_pack<E>(a[2], a[3])};
    }
}

// the largest over the wave's lanes: prefix maxima inside rows of 16 lanes, then lane 15 of one row to the next, then lane 31 to the upper half
__device__ __forceinline__ int win_wave_max(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xa, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}

// The rows (r = i G + g) that see a key: [lo, hi), and all of them behind lo when it is a sink
struct WinRun { int lo, hi; };
__device__ __forceinline__ WinRun win_key_rows(const WinDesc& d, const WinSeq& s, int key) {
  WinRun r;
  r.lo = (d.right < 0 ? 0 : max(0, key - d.right - s.shift)) * d.G;
  r.hi = (d.left < 0 || key < d.sinks ? s.qlen : max(0, min(s.qlen, key + d.left - s.shift + 1))) * d.G;
  if (key >= s.klen) r.hi = 0;
  return r;
}

// How the rows that see a tile of BK keys are shared out.  The first `nsink` tiles hold sinks, which EVERY later row sees: alone they would run as long as all
// rows are, 320 tiles of rows against 66 at 20,480 tokens and a window of 4097.  So their rows go to c1 workgroups, the other tiles' to c2 (1 unless there are too
// few tiles to fill the chip); a tile's workgroups leave their fp32 sums in the workspace and a second launch adds them in order.
struct WinSplit {
  int tiles, nsink, c1, c2, units;  // units: workgroups of one key head
  int fixed;                        // the rows of a tile of 64 lie at 32-bit distances from its first, the same in every tile
  float* part;                      // [B, Hk][slots][dK | dV][BK keys][DP]
};
__device__ __host__ __forceinline__ int win_split_slots(const WinSplit& s) { return (s.c1 > 1 ? s.nsink * s.c1 : 0) + (s.c2 > 1 ? (s.tiles - s.nsink) * s.c2 : 0); }

// Heads wider than 64 keep 192 registers of accumulators and of K and V: one wave a SIMD with all the registers, reading its operands ahead of their products,
// beats both two waves that spill (1164 us against 696 for a pass at 4 x 4093 tokens, 16 heads on 4 of 128) and workgroups of their own for dK and dV, which form S twice.
template <class E, int DP, int NW, int NS>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DP == 128 ? 1 : 2, DP == 128 ? 1 : 2))) void win_dkv_kernel(WinDesc d, WinRows wrows, WinSplit sp) {
  constexpr int KS = DP / 16, DT = DP / 32, IMG = 64 * DP * 2, BK = 32 * NW, SLOT = 2 * IMG, STAT = NS * SLOT;   // STAT: where the rows' numbers lie
  constexpr bool AHEAD = DP == 128;   // see the forward
  __shared__ __attribute__((aligned(16))) unsigned char smem[NS * (SLOT + 4 * 256)];   // slots of Q | dO, then of LSE | delta | exponent | spare
  using v8 = typename E::v8;
  using Copy = WinCopy<DP, NW>;
  const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), r31 = l & 31, h2 = l >> 5;
  int unit, hk, b;
  win_block_order(sp.units, d.Hk, d.B, unit, hk, b);
  const bool sink = unit < sp.nsink * sp.c1;
  const int c12 = sink ? sp.c1 : sp.c2, rest = sink ? unit : unit - sp.nsink * sp.c1, tile = (sink ? 0 : sp.nsink) + rest / c12, share = rest % c12;
  const WinSeq seq = win_seq(d, b);
  const int k0 = tile * BK, kw0 = k0 + 32 * w, key = kw0 + r31;
  int rlo = 0, rhi = 0;
  if (k0 < seq.klen) {
    rlo = win_key_rows(d, seq, k0).lo;
    rhi = k0 < d.sinks ? seq.qlen * d.G : win_key_rows(d, seq, min(k0 + BK, seq.klen) - 1).hi;
    if (rhi < rlo) rhi = rlo;
  }
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
    asm volatile("" : "+v"(x), "+v"(y));
    kf[ks] = __builtin_bit_cast(v8, x);
    vf[ks] = __builtin_bit_cast(v8, y);
  }
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int x = 0; x < 16; x++) { dk[dt][x] = 0.f; dv[dt][x] = 0.f; }
  int emax = WIN_NO_EXP, emin = WIN_NO_EXP;   // the exponent of this lane's key, and the least of the wave's keys
  const Copy copy(w, l, d.D);
  unsigned qoff[Copy::NP], goff[Copy::NP];
#pragma unroll
  for (int p = 0; p < Copy::NP; p++) {
    const int i = win_div(d, copy.row[p]), g = copy.row[p] - i * d.G;
    qoff[p] = (unsigned)(i * (unsigned)d.sq.r + g * (unsigned)d.sq.h) * 2 + copy.chunk[p] * 16;
    goff[p] = (unsigned)(i * (unsigned)d.sg.r + g * (unsigned)d.sg.h) * 2 + copy.chunk[p] * 16;
  }
  const uint16_t* qb = d.q + b * d.sq.b + (long long)hk * d.G * d.sq.h;
  const uint16_t* gb = d.g + b * d.sg.b + (long long)hk * d.G * d.sg.h;
  // the rows' numbers travel with the tile: wave 0 copies the LSEs, wave 1 the deltas, wave 2 the exponents (256 bytes; a count that is the same in all waves
  // wants a copy from each: the others' go to a slot nobody reads)
  const long long row0 = ((long long)b * d.Hk + hk) * d.Sq * d.G;
  const float* num = w == 1 ? wrows.ndelta + row0 : E::half && w == 2 ? (const float*)wrows.expo + row0 : wrows.lse2 + row0;
  const unsigned lds0 = __builtin_amdgcn_readfirstlane((int)lds_addr_of(smem)), lds = lds0 + w * (IMG / NW), lds_num = lds0 + STAT + 256 * min(w, 3);
  auto stage = [&](int j, int slot) __attribute__((always_inline)) {
    const int q0 = rlo + 64 * j;
    if (sp.fixed && q0 + 64 <= rhi) {
      const int i = win_div(d, q0);
      const uint16_t *qs = win_uniform(qb + (long long)i * d.sq.r), *gs = win_uniform(gb + (long long)i * d.sg.r);
#pragma unroll
      for (int p = 0; p < Copy::NP; p++) win_dma_off(qs, qoff[p], lds + slot * SLOT + p * 1024);
#pragma unroll
      for (int p = 0; p < Copy::NP; p++) win_dma_off(gs, goff[p], lds + slot * SLOT + IMG + p * 1024);
    } else {   // (a row past the last one: the last one, which is masked)
#pragma unroll
      for (int p = 0; p < Copy::NP; p++) {
        const int r = min(q0 + copy.row[p], rhi - 1), i = win_div(d, r);
        win_dma_ptr(qb + (long long)i * d.sq.r + (long long)(r - i * d.G) * d.sq.h + copy.chunk[p] * 8, lds + slot * SLOT + p * 1024);
        win_dma_ptr(gb + (long long)i * d.sg.r + (long long)(r - i * d.G) * d.sg.h + copy.chunk[p] * 8, lds + slot * SLOT + IMG + p * 1024);
      }
    }
    win_dma4_ptr(num + min(q0 + l, rhi - 1), lds_num + slot * 1024);
  };
  // rows that see this lane's key, and what this wave's keys see of a tile
  const WinRun mine = win_key_rows(d, seq, key);
  const int klast = min(kw0 + 32, seq.klen) - 1;
  const WinRun first = win_key_rows(d, seq, kw0), last = win_key_rows(d, seq, max(klast, 0));
  const int any_hi = min(rhi, kw0 < d.sinks ? seq.qlen * d.G : last.hi), all_lo = last.lo;
  const int all_hi = min(rhi, kw0 < d.sinks && klast >= d.sinks ? win_key_rows(d, seq, d.sinks).hi : first.hi);
  WinRead<DP> rd(lds0, l);
  auto rowtile = [&](int j, int off) __attribute__((always_inline)) {
    const int q0 = rlo + 64 * j;
    const unsigned char* st = smem + STAT + 1024 * (j % NS);
    if (kw0 > klast || q0 + 64 <= first.lo || q0 >= any_hi) return;   // nobody sees these keys
    const bool all = q0 >= all_lo && q0 + 64 <= all_hi;
    float unit = 1.f;
    if constexpr (E::half) {
      int er = *(const int*)(st + 512 + 4 * l);   // row q0 + l's
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(er > emin) != 0, 0)) {   // (seldom after the first tiles)
        const int a = max(0, min(64, mine.lo - q0)), z = max(0, min(64, min(mine.hi, rhi) - q0));
        const unsigned long long in = z > a ? (~0ull >> (64 - z + a)) << a : 0;   // the rows that this lane's key sees
        int e = emax;
        bool open = in != 0;
        // the tile's exponents from the largest down, until every key has met one of its rows (every turn takes a row out)
        for (int m = win_wave_max(er); m > WIN_NO_EXP && __builtin_amdgcn_ballot_w64(open) != 0; m = win_wave_max(er)) {
          if ((in & __builtin_amdgcn_ballot_w64(er == m)) != 0) { e = max(e, m); open = false; }
          if (er == m) er = WIN_NO_EXP;
        }
        if (__builtin_amdgcn_ballot_w64(e != emax && emax != WIN_NO_EXP) != 0) {   // (without an exponent nothing has been added yet)
          const float f = emax == WIN_NO_EXP ? 1.f : ldexpf(1.f, emax - e);
#pragma unroll
          for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int x = 0; x < 16; x++) dk[dt][x] *= f;
        }
        emax = e;
        emin = -win_wave_max(key < seq.klen ? -e : -INT_MAX);
      }
      unit = emax == WIN_NO_EXP ? 1.f : ldexpf(1.f, -emax);
    }
    // 32 rows at a time: qt's products over the channels, its P and dS, its products over the rows.  The matrix pipe runs beside the vector unit when their
    // instructions alternate (8 products and 64 others: 173 ns together, 125 and 115 alone, two waves a SIMD), so each half's vector work stands next to the other's products.
    f32x16 s[2], dp[2];
    u32x4 qa[2][KS], ga[2][KS];
    v8 pf[2][2], ds[2][2];
    s16x8 gc[2][2][DT], qc[2][2][DT];
    auto rows = [&](int qt) __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < KS; ks++) { qa[qt][ks] = rd.rows(ks, off + 64 * DP * qt); ga[qt][ks] = rd.rows(ks, off + IMG + 64 * DP * qt); }
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const f32x4 de = *(const f32x4*)(st + 256 + (32 * qt + 8 * x + 4 * h2) * 4);
#pragma unroll
        for (int y = 0; y < 4; y++) { s[qt][4 * x + y] = 0.f; dp[qt][4 * x + y] = de[y]; }
      }
    };
    auto scores = [&](int qt) __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        s[qt] = E::mfma(__builtin_bit_cast(v8, qa[qt][ks]), kf[ks], s[qt]);
        dp[qt] = E::mfma(__builtin_bit_cast(v8, ga[qt][ks]), vf[ks], dp[qt]);
      }
    };
    auto mask = [&](int qt) __attribute__((always_inline)) {
      const int o = q0 + 32 * qt + 4 * h2, lo = mine.lo - o, hi = min(mine.hi, rhi) - o;
#pragma unroll
      for (int x = 0; x < 16; x++) {
        const int r = (x & 3) + 8 * (x >> 2);
        const bool vis = r >= lo && r < hi;
        s[qt][x] = vis ? s[qt][x] : -INFINITY;
        dp[qt][x] = vis ? dp[qt][x] : 0.f;
      }
    };
    auto cols = [&](int qt) __attribute__((always_inline)) {
#pragma unroll
      for (int half = 0; half < 2; half++)
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
          gc[qt][half][dt] = rd.cols(dt, off + IMG + 64 * DP * qt + 32 * DP * half);
          qc[qt][half][dt] = rd.cols(dt, off + 64 * DP * qt + 32 * DP * half);
        }
    };
    auto probs = [&](int qt) __attribute__((always_inline)) {
#pragma unroll
      for (int x = 0; x < 16; x++) {
        const f32x4 ls = *(const f32x4*)(st + (32 * qt + 8 * (x >> 2) + 4 * h2) * 4);
        const float p = fast_exp2(__builtin_fmaf(s[qt][x], c, -ls[x & 3]));
        float g = p * dp[qt][x];
        if constexpr (E::half) g *= unit;
        pf[qt][x >> 3][x & 7] = (typename E::e)p;
        ds[qt][x >> 3][x & 7] = (typename E::e)g;
      }
      asm volatile("" : "+v"(pf[qt][0]), "+v"(pf[qt][1]), "+v"(ds[qt][0]), "+v"(ds[qt][1]));   // (here, not where they are first used)
    };
    auto grads = [&](int qt) __attribute__((always_inline)) {
#pragma unroll
      for (int half = 0; half < 2; half++)
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
          dv[dt] = E::mfma(__builtin_bit_cast(v8, gc[qt][half][dt]), pf[qt][half], dv[dt]);
          dk[dt] = E::mfma(__builtin_bit_cast(v8, qc[qt][half][dt]), ds[qt][half], dk[dt]);
        }
    };
    // Vector instructions behind a product: as many as probs has between them - but at one wave a SIMD, where both compete for issue, two beside the scores
    // (whose products the probabilities wait for) and six beside the gradients (4 x 4093 tokens, 16 heads on 4 of 128: 3 and 3 322 us, 4 and 4 313, 2 and 6 299)
    constexpr int VALU = E::half ? 72 : 56;
    rows(0);
    if constexpr (AHEAD) WIN_AHEAD();
    rows(1);
    scores(0);
    if (!all) mask(0);
    cols(0);
    scores(1);
    probs(0);
    win_weave<2 * KS, DP == 128 ? 2 : VALU / (2 * KS)>();
    if (!all) mask(1);
    cols(1);
    grads(0);
    probs(1);
    win_weave<4 * DT, DP == 128 ? 6 : VALU / (4 * DT)>();
    grads(1);
  };
  if (rlo < rhi) win_walk<NS, SLOT>((rhi - rlo + 63) / 64, win_arrived<(NS - 2) * (2 * Copy::NP + 1)>, stage, rowtile, [&](int by) { rd.move(by); });
  const float f = E::half && emax != WIN_NO_EXP ? ldexpf(d.scale, emax) : d.scale;
  if (c12 > 1) {   // [32-channel block][key][32 channels]: a lane's four channels go out as 16 bytes
    const int slot = sink || sp.c1 <= 1 ? rest : sp.nsink * sp.c1 + rest;
    float* part = sp.part + (((long long)b * d.Hk + hk) * win_split_slots(sp) + slot) * (2 * BK * DP);
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int rg = 0; rg < 4; rg++) {
        float* at = part + (dt * BK + 32 * w + r31) * 32 + 8 * rg + 4 * h2;
        *(f32x4*)at = (f32x4){dk[dt][4 * rg] * f, dk[dt][4 * rg + 1] * f, dk[dt][4 * rg + 2] * f, dk[dt][4 * rg + 3] * f};
        *(f32x4*)(at + BK * DP) = (f32x4){dv[dt][4 * rg], dv[dt][4 * rg + 1], dv[dt][4 * rg + 2], dv[dt][4 * rg + 3]};
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
      float a[4], g[4];
#pragma unroll
      for (int x = 0; x < 4; x++) { a[x] = live ? dk[dt][4 * rg + x] * f : 0.f; g[x] = live ? dv[dt][4 * rg + x] : 0.f; }
      *(u32x2*)(ok + d0) = (u32x2){el_pack<E>(a[0], a[1]), el_pack<E>(a[2], a[3])};
      *(u32x2*)(ov + d0) = (u32x2){el_pack<E>(g[0], g[1]), el_pack<E>(g[2], g[3])};
    }
}

// adds the shares of the tiles that were split: a workgroup takes 1024 / DP keys of one tile's dK or dV
template <class E, int DP, int BK>
__global__ __launch_bounds__(256) void win_dkv_join_kernel(WinDesc d, WinSplit sp) {
  constexpr int PER = DP / 4, KEYS = 256 / PER;   // four channels a thread
  const int split0 = sp.c1 > 1 ? 0 : sp.nsink, ntile = (sp.c2 > 1 ? sp.tiles : sp.nsink) - split0;   // the tiles [split0, split0 + ntile) were split
  const int groups = BK / KEYS;
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
  const int kl = kg * KEYS + threadIdx.x / PER, ch = (threadIdx.x % PER) * 4, key = tile * BK + kl;
  if (key >= d.Sk || ch >= d.D) return;
  const float* from = sp.part + (((long long)b * d.Hk + hk) * win_split_slots(sp) + slot0) * (2 * BK * DP) + part * BK * DP + ((ch >> 5) * BK + kl) * 32 + (ch & 31);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < c12; i++) s += *(const f32x4*)(from + (long long)i * (2 * BK * DP));
  if (key >= win_seq(d, b).klen) s = (f32x4){0.f, 0.f, 0.f, 0.f};
  const WinStride& st = part ? d.sdv : d.sdk;
  *(u32x2*)((part ? d.dv : d.dk) + b * st.b + key * st.r + hk * st.h + ch) = (u32x2){el_pack<E>(s[0], s[1]), el_pack<E>(s[2], s[3])};
}

static constexpr int WIN_BK = 128;   // keys a workgroup (4 waves of 32)
static int win_dp(const WinDesc& d) { return d.D <= 32 ? 32 : d.D <= 64 ? 64 : 128; }
// (a tile that starts at a whole query; long head-major operands have their heads further apart than 32 bits reach)
static bool win_fixed(const WinDesc& d, const WinStride& s) {
  return 64 % d.G == 0 && (64 / d.G - 1) * s.r + (d.G - 1) * s.h < (1ll << 30) - 128;
}
static WinSplit win_split(const WinDesc& d) {
  WinSplit s = {};
  s.fixed = win_fixed(d, d.sq) && win_fixed(d, d.sg);
  const int bk = WIN_BK;
  s.tiles = (d.Sk + bk - 1) / bk;
  s.nsink = d.left < 0 ? 0 : std::min(s.tiles, (int)(((long long)std::min(d.sinks, d.Sk) + bk - 1) / bk));
  // rows that see a tile: all (a sink, an open window to the left), or those of a window
  const long long all = (long long)d.Sq * d.G, window = d.left < 0 || d.right < 0 ? all : std::min<long long>(all, ((long long)d.left + d.right + bk) * d.G);
  const long long plain = (long long)(s.tiles - s.nsink) * d.Hk * d.B;
  // A share costs its sums' way through memory (128 KiB at 128 keys of 128 channels, out and back) and saves a part of its tile's rows, a microsecond or two for
  // 64 of them: no share has less than 1024 rows, and tiles are split only as far as there is room for more workgroups (counted as two a CU, though one fits at
  // 128 channels; the sinks' four)
  s.c2 = (int)std::max<long long>(1, std::min<long long>({512 / std::max<long long>(plain, 1), window / 1024, 64}));
  const long long share = std::max<long long>(1024, (window + s.c2 - 1) / s.c2), sinks = (long long)s.nsink * d.Hk * d.B;
  s.c1 = (int)std::max<long long>(1, std::min<long long>({(all + share - 1) / share, 1024 / std::max<long long>(sinks, 1), 64}));
  if (s.nsink == s.tiles) s.c2 = 1;
  if (s.nsink == 0) s.c1 = 1;
  s.units = s.nsink * s.c1 + (s.tiles - s.nsink) * s.c2;
  return s;
}
static size_t win_split_bytes(const WinDesc& d, const WinSplit& s) {
  return (size_t)win_split_slots(s) * d.Hk * d.B * 2 * WIN_BK * win_dp(d) * sizeof(float);
}

// workspace: the rows' LSE and -delta fp32 [B, Hk, Sq G] | exponents int32 [B, Hk, Sq G] (fp16) | the shares of split key tiles
static size_t win_rows_bytes(const WinDesc& d) { return ((size_t)d.B * d.H * d.Sq * 4 + 255) & ~(size_t)255; }
size_t window_attention_bwd_workspace_bytes(const WinDesc& d, int dtype) {
  if (window_attention_check(d, true, "window_attention_bwd", true)) return 0;
  return win_rows_bytes(d) * (dtype ? 3 : 2) + win_split_bytes(d, win_split(d)) + 256;
}

template <class E>
static int win_bwd(const WinDesc& d, void* ws, hipStream_t st) {
  const size_t nb = win_rows_bytes(d);
  const WinRows wr = {(float*)ws, (float*)((char*)ws + nb), E::half ? (int*)((char*)ws + 2 * nb) : nullptr};
  const long long n = (long long)d.B * d.H * d.Sq, rows = (long long)d.Sq * d.G, heads = (long long)d.Hk * d.B;
  if (n > 0) {
#define GO(DP) hipLaunchKernelGGL((win_rows_kernel<E, DP>), dim3((unsigned)((n + 2048 / DP - 1) / (2048 / DP))), dim3(256), 0, st, d, wr)
    if (d.D <= 32) GO(32);
    else if (d.D <= 64) GO(64);
    else GO(128);
#undef GO
#define GO(DP, NW, NS, OCC) hipLaunchKernelGGL((win_dq_kernel<E, DP, NW, NS, OCC>), dim3((unsigned)((rows + 32 * NW - 1) / (32 * NW) * heads)), dim3(64 * NW), 0, st, d, wr)
    if (d.D <= 32) GO(32, 4, 3, 3);
    else if (d.D <= 64) GO(64, 4, 3, 3);
    else GO(128, 4, 2, 2);
#undef GO
  }
  if (d.Sk > 0) {
    WinSplit sp = win_split(d);
    sp.part = (float*)((char*)ws + nb * (E::half ? 3 : 2));
    const dim3 grid((unsigned)(heads * sp.units));
    const int ntile = (sp.c1 > 1 ? sp.nsink : 0) + (sp.c2 > 1 ? sp.tiles - sp.nsink : 0);
#define GO(DP, NW, NS)                                                                                                                          \
  {                                                                                                                                                    \
    hipLaunchKernelGGL((win_dkv_kernel<E, DP, NW, NS>), grid, dim3(64 * NW), 0, st, d, wr, sp);                                                \
    if (ntile) hipLaunchKernelGGL((win_dkv_join_kernel<E, DP, 32 * NW>), dim3((unsigned)(2 * (32 * NW / (1024 / DP)) * ntile * heads)), dim3(256), 0, st, d, sp); \
  }
    if (d.D <= 32) GO(32, 4, 4)
    else if (d.D <= 64) GO(64, 4, 4)
    else GO(128, 4, 4)
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
