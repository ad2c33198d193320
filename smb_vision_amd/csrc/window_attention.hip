// Windowed attention with sinks, forward (window_attention.h has the definition).
//
// One workgroup owns 128 rows (4 waves x 32) of one key head and walks the run of keys that they see in tiles of 64, with the running maximum and sum of
// the softmax in 32 bits:
//   S^T[key][row] = K Q^T       matrix product 32x32x16: A = K from LDS, B = Q in registers.  The row sits on the lane, so maximum and sum are lane-local
//                               (one exchange between the wave's halves a tile)
//   O^T[d][row]  += V^T P^T     the accumulator of S^T, exponentiated and rounded to the type of V, IS the B operand; A = V^T by transposed LDS reads
// The scores are scaled in 32 bits behind the product (Q is not rounded a second time).  P is rounded to 16 bits for the second product, relative to its
// row's maximum; its sum is taken before the rounding, in 32 bits.
#include "window_attention.h"
#include <math.h>

namespace smbv {

static constexpr float WIN_THR = 6.f;  // log2 units

// A call whose row tiles do not fill the chip shares their runs of keys out as well: every share leaves its maximum (log2 units), its sum and its unnormalised O,
// and win_join_kernel joins them, always in the same order.
// part: [shares][B, Hk][tiles of 32 rows], each [DP / 32][32 rows][32 channels] of O, then [32 rows] pairs of maximum and sum
struct WinShares { int n; float* part; };
template <int DP> __device__ __forceinline__ float* win_part(const WinDesc& d, const WinShares& sh, int share, int b, int hk, int tile32, int tiles32) {
  return sh.part + ((((long long)share * d.B + b) * d.Hk + hk) * tiles32 + tile32) * (32 * (DP + 2));
}

// NW waves of 32 rows; NS slots of a K and a V tile
template <class E, int DP, int NW, int NS, int OCC>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void win_fwd_kernel(WinDesc d, WinShares sh) {
  constexpr int KS = DP / 16, DT = DP / 32, IMG = 64 * DP * 2, BM = 32 * NW;
  // Wide heads have two waves a SIMD and registers to spare: all of a tile's K operands and the first half of V's are read before the products that take them
  // (207 -> 191 us at 4 x 4093 tokens, 16 heads of 128, window 1024; at 64 channels three waves a SIMD hide the reads as well)
  constexpr bool AHEAD = DP == 128;
  using v8 = typename E::v8;
  using Copy = WinCopy<DP, NW>;
  __shared__ __attribute__((aligned(16))) unsigned char smem[NS * 2 * IMG];
  const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), r31 = l & 31, h2 = l >> 5;
  int tile, hk, b;
  win_block_order((int)(((long long)d.Sq * d.G + BM - 1) / BM) * sh.n, d.Hk, d.B, tile, hk, b);
  const int share = tile % sh.n;
  tile /= sh.n;
  const WinSeq seq = win_seq(d, b);
  const int r0 = tile * BM, rows = d.Sq * d.G;
  const int i0 = win_div(d, r0), i1 = min(seq.qlen, win_div(d, min(r0 + BM, rows) - 1) + 1);
  const WinKeys wk = win_keys(d, seq, i0, i1);
  const int r = r0 + 32 * w + r31, i = win_div(d, r), head = hk * d.G + (r - i * d.G);
  const bool live = r < rows && i < seq.qlen;
  const WinView view = win_view(d, seq, wk, i);
  const uint16_t* kb = d.k + b * d.sk.b + hk * d.sk.h;
  const uint16_t* vb = d.v + b * d.sv.b + hk * d.sv.h;
  const Copy copy(w, l, d.D);
  unsigned koff[Copy::NP], voff[Copy::NP];
  copy.offsets(koff, d.sk.r);
  copy.offsets(voff, d.sv.r);
  const unsigned lds = __builtin_amdgcn_readfirstlane((int)(lds_addr_of(smem) + w * (IMG / NW)));
  const long long all = (wk.n + 63) / 64;
  const int t0 = (int)(all * share / sh.n), nt = (int)(all * (share + 1) / sh.n) - t0;   // this share's tiles
  auto stage = [&](int j, int slot) __attribute__((always_inline)) {
    copy.keys(kb, d.sk.r, koff, wk, 64 * (t0 + j), lds + slot * 2 * IMG);
    copy.keys(vb, d.sv.r, voff, wk, 64 * (t0 + j), lds + slot * 2 * IMG + IMG);
  };
  v8 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    u32x4 x = {0, 0, 0, 0};
    if (live && 16 * ks + 8 * h2 < d.D) x = *(const u32x4*)(d.q + b * d.sq.b + i * d.sq.r + head * d.sq.h + 16 * ks + 8 * h2);
    asm volatile("" : "+v"(x));   // (waited for here, not in the loop)
    qf[ks] = __builtin_bit_cast(v8, x);
  }
  f32x16 ot[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int x = 0; x < 16; x++) ot[dt][x] = 0.f;
  float m2 = -INFINITY, sum = 0.f;
  const float c = d.scale * 1.4426950408889634f;
  // this wave's first and last query
  const int wi0 = win_div(d, r0 + 32 * w), wi1 = min(seq.qlen, win_div(d, min(r0 + 32 * w + 32, rows) - 1) + 1);
  const WinView v0 = win_view(d, seq, wk, wi0), v1 = win_view(d, seq, wk, wi1 - 1);
  WinRead<DP> rd(lds_addr_of(smem), l);
  auto keys = [&](int j, int off) __attribute__((always_inline)) {
    const int kind = wi0 < wi1 ? win_tile(v0, v1, 64 * (t0 + j)) : WIN_NONE;
    if (kind == WIN_NONE) return;
    f32x16 sc[2];
    u32x4 kf[2][KS];
    if constexpr (AHEAD) {
#pragma unroll
      for (int x = 0; x < 2 * KS; x++) kf[x / KS][x % KS] = rd.rows(x % KS, off + 64 * DP * (x / KS));
      WIN_AHEAD();
    }
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
#pragma unroll
      for (int x = 0; x < 16; x++) sc[kt][x] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        if constexpr (!AHEAD) kf[kt][ks] = rd.rows(ks, off + 64 * DP * kt);
        sc[kt] = E::mfma(__builtin_bit_cast(v8, kf[kt][ks]), qf[ks], sc[kt]);
      }
    }
    if (kind != WIN_ALL) {
#pragma unroll
      for (int kt = 0; kt < 2; kt++) win_mask(sc[kt], kind, view, 64 * (t0 + j) + 32 * kt + 4 * h2);
    }
    float mx = fmaxf(sc[0][0], sc[1][0]);
#pragma unroll
    for (int x = 1; x < 16; x++) mx = fmaxf(fmaxf(mx, sc[0][x]), sc[1][x]);
    mx = win_halves_max(mx) * c;
    // the running reference moves only when a score outgrows it by 2^THR: exp2 stays in range of the 16-bit P (and P keeps its relative precision)
    if (__builtin_amdgcn_ballot_w64(mx > m2 + WIN_THR) != 0) {
      const float m_new = fmaxf(m2, mx);
      const float alpha = m2 == m_new ? 1.f : fast_exp2(m2 - m_new);   // (m2 = -inf: nothing is accumulated yet)
      m2 = m_new;
      sum *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int x = 0; x < 16; x++) ot[dt][x] *= alpha;
    }
    const float ref = m2 == -INFINITY ? 0.f : m2;
    s16x8 vf[4][DT];
    if constexpr (AHEAD) {   // V two 16-key steps ahead
#pragma unroll
      for (int x = 0; x < 2 * DT; x++) vf[x / DT][x % DT] = rd.cols(x % DT, off + IMG + 32 * DP * (x / DT));
      WIN_AHEAD();
    }
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
      v8 pf;
#pragma unroll
      for (int x = 0; x < 8; x++) {
        const float p = fast_exp2(__builtin_fmaf(sc[ks >> 1][8 * (ks & 1) + x], c, -ref));
        sum += p;
        pf[x] = (typename E::e)p;
      }
#pragma unroll
      for (int dt = 0; dt < DT; dt++) {
        if constexpr (!AHEAD) vf[ks][dt] = rd.cols(dt, off + IMG + 32 * DP * ks);
        ot[dt] = E::mfma(__builtin_bit_cast(v8, vf[ks][dt]), pf, ot[dt]);
      }
      if (AHEAD && ks < 2) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++) vf[ks + 2][dt] = rd.cols(dt, off + IMG + 32 * DP * (ks + 2));
      }
    }
  };
  if (nt > 0) win_walk<NS, 2 * IMG>(nt, win_arrived<(NS - 2) * 2 * Copy::NP>, stage, keys, [&](int by) { rd.move(by); });
  sum = win_halves_sum(sum);
  if (sh.n > 1) {
    const int tiles = (rows + 31) / 32;
    if (r0 + 32 * w >= rows) return;
    float* out = win_part<DP>(d, sh, share, b, hk, tile * NW + w, tiles);
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int rg = 0; rg < 4; rg++)
        if (32 * dt + 8 * rg < d.D) *(f32x4*)(out + (dt * 32 + r31) * 32 + 8 * rg + 4 * h2) = (f32x4){ot[dt][4 * rg], ot[dt][4 * rg + 1], ot[dt][4 * rg + 2], ot[dt][4 * rg + 3]};
    if (h2 == 0) *(float2*)(out + 32 * DP + 2 * r31) = make_float2(m2, sum);
    return;
  }
  const bool some = live && sum != 0.f;   // (a row that sees nothing is 0, also beside an infinity in a value that others see)
  const float inv = 1.0f / sum;
  if (r >= rows) return;
  const long long oo = b * d.so.b + i * d.so.r + head * d.so.h;
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int rg = 0; rg < 4; rg++) {
      const int d0 = 32 * dt + 8 * rg + 4 * h2;
      if (d0 >= d.D) continue;
      float f[4];
#pragma unroll
      for (int x = 0; x < 4; x++) f[x] = some ? ot[dt][4 * rg + x] * inv : 0.f;
      const u32x2 pk = {el_pack<E>(f[0], f[1]), el_pack<E>(f[2], f[3])};
      *(u32x2*)(d.o + oo + d0) = pk;
      if (d.o_lo) {
#pragma unroll
        for (int x = 0; x < 4; x++) f[x] -= el_f<E>((uint16_t)(pk[x >> 1] >> (16 * (x & 1))));
        *(u32x2*)(d.o_lo + oo + d0) = (u32x2){el_pack<E>(f[0], f[1]), el_pack<E>(f[2], f[3])};
      }
    }
  if (h2 == 0) d.lse[((long long)b * d.H + head) * d.Sq + i] = !some ? -INFINITY : (m2 + __log2f(sum)) * 0.6931471805599453f;
}

// ---- few rows against many keys (single tokens) ------------------------------------------------------------------------------------------------------------
// Bound by HBM: every key and value is read once for a handful of rows.  A workgroup takes 32 rows of one key head and a share of their run of keys; its four
// waves take 32-key tiles in turn, each with a ring of its own, so nobody waits for anybody until their sums are joined in LDS.  (16 single tokens on caches of
// 16,384 keys, 8 key heads of 128, window 8192: 216 us by the 128-row kernel, one wave of which has rows; 110 us, 4.8 TB/s, here.)
// a row's N channels from ch0 on: O normalised, its residual, and by the first of the row's threads the LSE
template <class E, int N>
__device__ __forceinline__ void win_few_store(const WinDesc& d, const float (&o)[N], int ch0, int rr, int hk, int b, float m, float total, const WinSeq& seq) {
  const int i = win_div(d, rr), head = hk * d.G + (rr - i * d.G);
  const bool some = i < seq.qlen && total != 0.f;
  const float inv = 1.0f / total;
  const long long oo = b * d.so.b + i * d.so.r + head * d.so.h + ch0;
#pragma unroll
  for (int x = 0; x < N; x += 4) {
    if (ch0 + x >= d.D) continue;
    float f[4];
#pragma unroll
    for (int y = 0; y < 4; y++) f[y] = some ? o[x + y] * inv : 0.f;
    const u32x2 pk = {el_pack<E>(f[0], f[1]), el_pack<E>(f[2], f[3])};
    *(u32x2*)(d.o + oo + x) = pk;
    if (d.o_lo) {
#pragma unroll
      for (int y = 0; y < 4; y++) f[y] -= el_f<E>((uint16_t)(pk[y >> 1] >> (16 * (y & 1))));
      *(u32x2*)(d.o_lo + oo + x) = (u32x2){el_pack<E>(f[0], f[1]), el_pack<E>(f[2], f[3])};
    }
  }
  if (ch0 == 0) d.lse[((long long)b * d.H + head) * d.Sq + i] = !some ? -INFINITY : (m + __log2f(total)) * 0.6931471805599453f;
}

template <class E, int DP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 4))) void win_few_kernel(WinDesc d, WinShares sh) {
  constexpr int KS = DP / 16, DT = DP / 32, IMG = 32 * DP * 2, NS = DP == 32 ? 3 : 2, RING = NS * 2 * IMG, NP = IMG / 1024, R = 512 / DP, C = DP / 8;
  using v8 = typename E::v8;
  constexpr int JOIN = 4 * 32 * (DP + 4) * 4;   // the waves' O (rows of DP + 4 floats: the 16-byte pieces of a row fall on different banks), maximum, sum
  __shared__ __attribute__((aligned(16))) unsigned char smem[4 * RING > JOIN ? 4 * RING : JOIN];
  const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), r31 = l & 31, h2 = l >> 5;
  const int rows = d.Sq * d.G, tiles = (rows + 31) / 32;
  int unit, hk, b;
  win_block_order(tiles * sh.n, d.Hk, d.B, unit, hk, b);
  const int tile = unit / sh.n, share = unit - tile * sh.n;
  const WinSeq seq = win_seq(d, b);
  const int r0 = tile * 32, i0 = win_div(d, r0), i1 = min(seq.qlen, win_div(d, min(r0 + 32, rows) - 1) + 1);
  const WinKeys wk = win_keys(d, seq, i0, i1);
  const int r = r0 + r31, i = win_div(d, r), head = hk * d.G + (r - i * d.G);
  const bool live = r < rows && i < seq.qlen;
  const WinView view = win_view(d, seq, wk, i), v0 = win_view(d, seq, wk, i0), v1 = win_view(d, seq, wk, i1 - 1);
  const uint16_t* kb = d.k + b * d.sk.b + hk * d.sk.h;
  const uint16_t* vb = d.v + b * d.sv.b + hk * d.sv.h;
  // this share's tiles of 32 keys [t0, t1), this wave's: t0 + w, t0 + w + 4, ...
  const long long nt = (wk.n + 31) / 32;
  const int t0 = (int)(nt * share / sh.n), t1 = (int)(nt * (share + 1) / sh.n), mine = t1 - t0 > w ? (t1 - t0 - w + 3) / 4 : 0;
  const unsigned lds = __builtin_amdgcn_readfirstlane((int)(lds_addr_of(smem) + w * RING));
  auto stage = [&](int j, int slot) __attribute__((always_inline)) {
    const int u0 = 32 * (t0 + w + 4 * j);
#pragma unroll
    for (int p = 0; p < NP; p++) {
      const int row = p * R + l / C, chunk = min((win_img<DP>(row, l % C) - row * DP * 2) >> 4, d.D / 8 - 1), u = min(u0 + row, wk.n - 1);
      const long long key = u < wk.ns ? u : u + wk.jump;
      win_dma_ptr(kb + key * d.sk.r + chunk * 8, lds + slot * 2 * IMG + p * 1024);
      win_dma_ptr(vb + key * d.sv.r + chunk * 8, lds + slot * 2 * IMG + IMG + p * 1024);
    }
  };
  if (mine > 0) {
#pragma unroll
    for (int s = 0; s < NS - 1; s++) stage(s, s);
  }
  v8 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    u32x4 x = {0, 0, 0, 0};
    if (live && 16 * ks + 8 * h2 < d.D) x = *(const u32x4*)(d.q + b * d.sq.b + i * d.sq.r + head * d.sq.h + 16 * ks + 8 * h2);
    asm volatile("" : "+v"(x));
    qf[ks] = __builtin_bit_cast(v8, x);
  }
  f32x16 ot[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int x = 0; x < 16; x++) ot[dt][x] = 0.f;
  float m2 = -INFINITY, sum = 0.f;
  const float c = d.scale * 1.4426950408889634f;
  const WinRead<DP> rd(lds, l);
  for (int j = 0; j < mine; j += NS) {
#pragma unroll
    for (int s = 0; s < NS; s++) {
      if (j + s >= mine) break;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (this wave's reads of the slot that is filled next have returned)
      stage(j + s + NS - 1, (s + NS - 1) % NS);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * 2 * NP) : "memory");
      const int off = s * 2 * IMG, u0 = 32 * (t0 + w + 4 * (j + s));
      f32x16 sc;
#pragma unroll
      for (int x = 0; x < 16; x++) sc[x] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) sc = E::mfma(__builtin_bit_cast(v8, rd.rows(ks, off)), qf[ks], sc);
      const int kind = win_tile<32>(v0, v1, u0);
      if (kind != WIN_ALL) win_mask(sc, kind == WIN_NONE ? WIN_UPPER | WIN_LOWER | WIN_SINKS : kind, view, u0 + 4 * h2);
      float mx = sc[0];
#pragma unroll
      for (int x = 1; x < 15; x += 2) mx = fmaxf(fmaxf(mx, sc[x]), sc[x + 1]);
      mx = win_halves_max(fmaxf(mx, sc[15])) * c;
      if (__builtin_amdgcn_ballot_w64(mx > m2 + WIN_THR) != 0) {
        const float m_new = fmaxf(m2, mx), alpha = m2 == m_new ? 1.f : fast_exp2(m2 - m_new);
        m2 = m_new;
        sum *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int x = 0; x < 16; x++) ot[dt][x] *= alpha;
      }
      const float ref = m2 == -INFINITY ? 0.f : m2;
#pragma unroll
      for (int ks = 0; ks < 2; ks++) {
        v8 pf;
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const float p = fast_exp2(__builtin_fmaf(sc[8 * ks + x], c, -ref));
          sum += p;
          pf[x] = (typename E::e)p;
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) ot[dt] = E::mfma(__builtin_bit_cast(v8, rd.cols(dt, off + IMG + 32 * DP * ks)), pf, ot[dt]);
      }
    }
  }
  win_drain();
  sum = win_halves_sum(sum);
  __syncthreads();
  // join the four waves: row r31's O in LDS [wave][row][DP + 4], then its maximum and sum
  float* join = (float*)smem;
  constexpr int LD = DP + 4;
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int rg = 0; rg < 4; rg++)
      *(f32x4*)(join + (w * 32 + r31) * LD + 32 * dt + 8 * rg + 4 * h2) = (f32x4){ot[dt][4 * rg], ot[dt][4 * rg + 1], ot[dt][4 * rg + 2], ot[dt][4 * rg + 3]};
  if (h2 == 0) { join[(w * 32 + r31) * LD + DP] = m2; join[(w * 32 + r31) * LD + DP + 1] = sum; }
  __syncthreads();
  const int row = t >> 3, ch0 = (t & 7) * (DP / 8);   // 8 threads a row
  const float* mr = join + row * LD + DP;
  float m = -INFINITY, wgt[4], total = 0.f;
#pragma unroll
  for (int x = 0; x < 4; x++) m = fmaxf(m, mr[x * 32 * LD]);
#pragma unroll
  for (int x = 0; x < 4; x++) {
    wgt[x] = m == -INFINITY ? 0.f : fast_exp2(mr[x * 32 * LD] - m);
    total += wgt[x] * mr[x * 32 * LD + 1];
  }
  float o[DP / 8];
#pragma unroll
  for (int x = 0; x < DP / 8; x += 4) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int y = 0; y < 4; y++) a += *(const f32x4*)(join + (y * 32 + row) * LD + ch0 + x) * wgt[y];
    o[x] = a[0]; o[x + 1] = a[1]; o[x + 2] = a[2]; o[x + 3] = a[3];
  }
  if (sh.n > 1) {
    float* out = win_part<DP>(d, sh, share, b, hk, tile, tiles);
#pragma unroll
    for (int x = 0; x < DP / 8; x += 4)
      if (ch0 + x < d.D) *(f32x4*)(out + (((ch0 + x) >> 5) * 32 + row) * 32 + ((ch0 + x) & 31)) = (f32x4){o[x], o[x + 1], o[x + 2], o[x + 3]};
    if (ch0 == 0) *(float2*)(out + 32 * DP + 2 * row) = make_float2(m, total);
    return;
  }
  const int rr = r0 + row;
  if (rr >= rows) return;
  win_few_store<E, DP / 8>(d, o, ch0, rr, hk, b, m, total, seq);
}

// 8 lanes a row's channels, SG groups of them its shares (8 where there are many: one after the other they took 31 us for 32 shares of 64 rows)
template <class E, int DP, int SG>
__global__ __launch_bounds__(256) void win_join_kernel(WinDesc d, WinShares sh) {
  const int rows = d.Sq * d.G, tiles = (rows + 31) / 32, l = threadIdx.x & (8 * SG - 1), ch0 = (l & 7) * (DP / 8);
  const long long x = (long long)blockIdx.x * (32 / SG) + threadIdx.x / (8 * SG);
  if (x >= (long long)rows * d.Hk * d.B) return;
  const int hb = (int)(x / rows), rr = (int)(x - (long long)hb * rows), hk = hb % d.Hk, b = hb / d.Hk, row = rr & 31;
  float m = -INFINITY, total = 0.f, o[DP / 8];
#pragma unroll
  for (int i = 0; i < DP / 8; i++) o[i] = 0.f;
  for (int s = l >> 3; s < sh.n; s += SG) {
    const float* at = win_part<DP>(d, sh, s, b, hk, rr >> 5, tiles);
    const float2 ms = *(const float2*)(at + 32 * DP + 2 * row);
    const float mn = fmaxf(m, ms.x), keep = m == -INFINITY ? 0.f : fast_exp2(m - mn), w = ms.x == -INFINITY ? 0.f : fast_exp2(ms.x - mn);
    m = mn;
    total = total * keep + w * ms.y;
#pragma unroll
    for (int i = 0; i < DP / 8; i += 4) {
      if (ch0 + i >= d.D) continue;
      const f32x4 p = *(const f32x4*)(at + (((ch0 + i) >> 5) * 32 + row) * 32 + ((ch0 + i) & 31));
#pragma unroll
      for (int y = 0; y < 4; y++) o[i + y] = o[i + y] * keep + w * p[y];
    }
  }
  float all = m;
#pragma unroll
  for (int k = 8; k < 8 * SG; k <<= 1) all = fmaxf(all, __shfl_xor(all, k, 64));
  const float w = m == -INFINITY ? 0.f : fast_exp2(m - all);
  total *= w;
#pragma unroll
  for (int k = 8; k < 8 * SG; k <<= 1) total += __shfl_xor(total, k, 64);
#pragma unroll
  for (int i = 0; i < DP / 8; i++) {
    o[i] *= w;
#pragma unroll
    for (int k = 8; k < 8 * SG; k <<= 1) o[i] += __shfl_xor(o[i], k, 64);
  }
  if (l < 8) win_few_store<E, DP / 8>(d, o, ch0, rr, hk, b, all, total, win_seq(d, b));
}

int window_attention_check(const WinDesc& d, bool backward, const char* what, bool sizes_only) {
  if (d.B < 0 || d.Sq < 0 || d.Sk < 0 || d.Hk <= 0 || d.H <= 0 || d.H % d.Hk) { set_error("%s: bad shape B=%d Sq=%d Sk=%d H=%d Hk=%d (H a multiple of Hk)", what, d.B, d.Sq, d.Sk, d.H, d.Hk); return SMBV_ERR_SHAPE; }
  if (d.D <= 0 || d.D > 128 || (d.D & 7)) { set_error("%s: head width %d (a multiple of 8 up to 128)", what, d.D); return SMBV_ERR_SHAPE; }
  if (d.Sk >= (1 << 29) || d.Sq >= (1 << 29) || (unsigned long long)d.Sq * d.G * d.G >= (1ull << 31)) { set_error("%s: Sq=%d Sk=%d with %d heads to a key head is too long for one call", what, d.Sq, d.Sk, d.G); return SMBV_ERR_SHAPE; }
  // a launch has fewer than 2^24 workgroups of 256: 32 rows or 128 keys of one head each, and one pass of the backward 8 lanes or more a row
  const unsigned long long most = 1ull << 24, heads = (unsigned long long)d.Hk * d.B;
  if (((unsigned long long)d.Sq * d.G + 31) / 32 * heads >= most || ((unsigned long long)d.Sk + 127) / 128 * heads >= most || (unsigned long long)d.B * d.H * d.Sq >= 16 * most) { set_error("%s: too many rows for one call", what); return SMBV_ERR_SHAPE; }
  if (!(d.scale > 0.f) || !(d.scale < INFINITY)) { set_error("%s: scale must be positive and finite", what); return SMBV_ERR_ARG; }
  if (d.sinks < 0) { set_error("%s: sinks must not be negative", what); return SMBV_ERR_ARG; }
  if (sizes_only) return SMBV_OK;
  const struct { const void* p; const WinStride* s; long long n; const char* name; bool need; int align; } t[] = {
      {d.q, &d.sq, d.Sq, "q", true, 16}, {d.k, &d.sk, d.Sk, "k", true, 16}, {d.v, &d.sv, d.Sk, "v", true, 16},
      {backward ? (const void*)d.o_in : d.o, &d.so, d.Sq, "o", true, 16}, {backward ? (const void*)d.o_lo_in : d.o_lo, &d.so, d.Sq, "o_lo", false, 16},
      {d.g, &d.sg, d.Sq, "d_o", backward, 16}, {d.dq, &d.sdq, d.Sq, "dq", backward, 16}, {d.dk, &d.sdk, d.Sk, "dk", backward, 16}, {d.dv, &d.sdv, d.Sk, "dv", backward, 16}};
  for (const auto& x : t) {
    if (!x.p) {
      if (x.need && x.n > 0 && d.B > 0) { set_error("%s: %s is null", what, x.name); return SMBV_ERR_ARG; }
      continue;
    }
    if (((uintptr_t)x.p & (x.align - 1)) || ((x.s->b | x.s->r | x.s->h) & 7)) { set_error("%s: %s must be 16-byte aligned with strides that are multiples of 8 elements", what, x.name); return SMBV_ERR_ALIGN; }
    // (rows of keys and values inside a tile are reached by 32-bit offsets; everything else by 64-bit ones, to any distance that memory has)
    if (x.s->r >= (x.s == &d.sk || x.s == &d.sv ? 1ll << 24 : 1ll << 40) || x.s->h >= (1ll << 40)) { set_error("%s: %s has its rows or heads too many elements apart", what, x.name); return SMBV_ERR_SHAPE; }
    if (x.s->b < 0 || x.s->r < 0 || x.s->h < 0) { set_error("%s: %s has a negative stride", what, x.name); return SMBV_ERR_SHAPE; }
  }
  if (!d.lse && d.B > 0 && d.Sq > 0) { set_error("%s: lse is null", what); return SMBV_ERR_ARG; }
  return SMBV_OK;
}

// Up to 64 rows a key head go to the 32-row kernel: at 128 rows most of a workgroup would have none.  Shares: as many as bring every CU the workgroups that it
// holds (by LDS and registers: one at 128 channels and few rows, else two or three), none with less than 256 (512) keys, which cost about what a share's sums do
// (two caches of 4001 keys, 16 heads on 4 of 80, window 1500, in a replayed graph: 12 queries, at least 128 keys a share 15.1 us, 256 14.8, 512 17.1;
// 333 queries, at least 256 keys 37.8 us, 512 33.7, 1024 41.6).
struct WinPlan { bool few; int shares; };
static WinPlan win_plan(const WinDesc& d) {
  const long long rows = (long long)d.Sq * d.G, heads = (long long)d.Hk * d.B;
  WinPlan p;
  p.few = rows <= 64;
  const int tile = p.few ? 32 : 128;
  const long long units = std::max<long long>(1, (rows + tile - 1) / tile * heads), room = p.few ? (d.D > 64 ? 256 : 512) : (d.D > 64 ? 512 : 768);
  long long keys = d.Sk;   // of a row tile at most
  if (d.left >= 0 && d.right >= 0) keys = std::min<long long>(keys, (long long)d.left + d.right + tile + d.sinks);
  p.shares = (int)std::max<long long>(1, std::min<long long>(room / units, keys / (p.few ? 256 : 512)));
  return p;
}
static size_t win_shares_bytes(const WinDesc& d) {
  const int dp = d.D <= 32 ? 32 : d.D <= 64 ? 64 : 128, n = win_plan(d).shares;
  return n > 1 ? (size_t)n * d.B * d.Hk * (((size_t)d.Sq * d.G + 31) / 32) * 32 * (dp + 2) * sizeof(float) : 0;
}

template <class E>
static int win_fwd(const WinDesc& d, void* ws, hipStream_t st) {
  const long long rows = (long long)d.Sq * d.G, heads = (long long)d.Hk * d.B;
  const WinPlan p = win_plan(d);
  const WinShares sh = {p.shares, (float*)ws};
  const dim3 few((unsigned)((rows + 31) / 32 * sh.n * heads)), many((unsigned)((rows + 127) / 128 * sh.n * heads)), join4((unsigned)((rows * heads + 3) / 4)), join32((unsigned)((rows * heads + 31) / 32));
#define GO(DP, NS, OCC)                                                                                                     \
  {                                                                                                                         \
    if (p.few) hipLaunchKernelGGL((win_few_kernel<E, DP>), few, dim3(256), 0, st, d, sh);                                   \
    else hipLaunchKernelGGL((win_fwd_kernel<E, DP, 4, NS, OCC>), many, dim3(256), 0, st, d, sh);                            \
    if (sh.n > 4) hipLaunchKernelGGL((win_join_kernel<E, DP, 8>), join4, dim3(256), 0, st, d, sh);                          \
    else if (sh.n > 1) hipLaunchKernelGGL((win_join_kernel<E, DP, 1>), join32, dim3(256), 0, st, d, sh);                    \
  }
  if (d.D <= 32) GO(32, 3, 4) else if (d.D <= 64) GO(64, 3, 3) else GO(128, 2, 2)
#undef GO
  return check_launch("window_attention_fwd");
}

// workspace: the shares' sums
size_t window_attention_fwd_workspace_bytes(const WinDesc& d) {
  if (window_attention_check(d, false, "window_attention_fwd", true)) return 0;
  const size_t n = win_shares_bytes(d);
  return n ? n + 256 : 0;
}

int window_attention_fwd(const WinDesc& d, int dtype, void* ws, size_t ws_bytes, hipStream_t st) {
  if (int rc = window_attention_check(d, false, "window_attention_fwd")) return rc;
  if (d.B == 0 || d.Sq == 0) return SMBV_OK;
  const size_t need = window_attention_fwd_workspace_bytes(d);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 255))) { set_error("window_attention_fwd: workspace short or not 256-byte aligned (%zu < %zu)", ws_bytes, need); return SMBV_ERR_WORKSPACE; }
  return dtype == 0 ? win_fwd<ElBf16>(d, ws, st) : win_fwd<ElF16>(d, ws, st);
}

}  // namespace smbv
