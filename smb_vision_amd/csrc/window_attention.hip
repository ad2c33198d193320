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

// NW waves of 32 rows; NS slots of a K and a V tile
template <class E, int DP, int NW, int NS, int OCC>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void win_fwd_kernel(WinDesc d) {
  constexpr int KS = DP / 16, DT = DP / 32, IMG = 64 * DP * 2, BM = 32 * NW;
  // Wide heads have two waves a SIMD and registers to spare: all of a tile's K operands and the first half of V's are read before the products that take them
  // (207 -> 191 us at 4 x 4093 tokens, 16 heads of 128, window 1024; at 64 channels three waves a SIMD hide the reads as well)
  constexpr bool AHEAD = DP == 128;
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
  const Copy copy(w, l, d.D);
  unsigned koff[Copy::NP], voff[Copy::NP];
  copy.offsets(koff, d.sk.r);
  copy.offsets(voff, d.sv.r);
  const unsigned lds = __builtin_amdgcn_readfirstlane((int)(lds_addr_of(smem) + w * (IMG / NW)));
  auto stage = [&](int j, int slot) __attribute__((always_inline)) {
    copy.keys(kb, d.sk.r, koff, wk, 64 * j, lds + slot * 2 * IMG);
    copy.keys(vb, d.sv.r, voff, wk, 64 * j, lds + slot * 2 * IMG + IMG);
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
  const int nt = (wk.n + 63) / 64;
  // this wave's first and last query
  const int wi0 = win_div(d, r0 + 32 * w), wi1 = min(seq.qlen, win_div(d, min(r0 + 32 * w + 32, rows) - 1) + 1);
  const WinView v0 = win_view(d, seq, wk, wi0), v1 = win_view(d, seq, wk, wi1 - 1);
  WinRead<DP> rd(lds_addr_of(smem), l);
  auto keys = [&](int j, int off) __attribute__((always_inline)) {
    const int kind = wi0 < wi1 ? win_tile(v0, v1, 64 * j) : WIN_NONE;
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
      for (int kt = 0; kt < 2; kt++) win_mask(sc[kt], kind, view, 64 * j + 32 * kt + 4 * h2);
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
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
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
      for (int x = 0; x < 4; x++) f[x] = live ? ot[dt][4 * rg + x] * inv : 0.f;
      const u32x2 pk = {el_pack<E>(f[0], f[1]), el_pack<E>(f[2], f[3])};
      *(u32x2*)(d.o + oo + d0) = pk;
      if (d.o_lo) {
#pragma unroll
        for (int x = 0; x < 4; x++) f[x] -= el_f<E>((uint16_t)(pk[x >> 1] >> (16 * (x & 1))));
        *(u32x2*)(d.o_lo + oo + d0) = (u32x2){el_pack<E>(f[0], f[1]), el_pack<E>(f[2], f[3])};
      }
    }
  if (h2 == 0) d.lse[((long long)b * d.H + head) * d.Sq + i] = !live || sum == 0.f ? -INFINITY : (m2 + __log2f(sum)) * 0.6931471805599453f;
}

int window_attention_check(const WinDesc& d, bool backward, const char* what, bool sizes_only) {
  if (d.B < 0 || d.Sq < 0 || d.Sk < 0 || d.Hk <= 0 || d.H <= 0 || d.H % d.Hk) { set_error("%s: bad shape B=%d Sq=%d Sk=%d H=%d Hk=%d (H a multiple of Hk)", what, d.B, d.Sq, d.Sk, d.H, d.Hk); return SMBV_ERR_SHAPE; }
  if (d.D <= 0 || d.D > 128 || (d.D & 7)) { set_error("%s: head width %d (a multiple of 8 up to 128)", what, d.D); return SMBV_ERR_SHAPE; }
  if (d.Sk >= (1 << 29) || d.Sq >= (1 << 29) || (unsigned long long)d.Sq * d.G * d.G >= (1ull << 31)) { set_error("%s: Sq=%d Sk=%d with %d heads to a key head is too long for one call", what, d.Sq, d.Sk, d.G); return SMBV_ERR_SHAPE; }
  if (((unsigned long long)d.Sq * d.G + 63) / 64 * d.Hk * d.B >= (1ull << 30) || ((unsigned long long)d.Sk + 127) / 128 * d.Hk * d.B >= (1ull << 30) || (unsigned long long)d.B * d.H * d.Sq >= (1ull << 40)) { set_error("%s: too many rows for one call", what); return SMBV_ERR_SHAPE; }
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
    if (x.s->r >= (1 << 24) || x.s->h >= (1 << 24)) { set_error("%s: %s has rows or heads 2^24 elements apart", what, x.name); return SMBV_ERR_SHAPE; }   // (offsets inside a tile are 32-bit)
    if (x.s->b < 0 || x.s->r < 0 || x.s->h < 0) { set_error("%s: %s has a negative stride", what, x.name); return SMBV_ERR_SHAPE; }
  }
  if (!d.lse && d.B > 0 && d.Sq > 0) { set_error("%s: lse is null", what); return SMBV_ERR_ARG; }
  return SMBV_OK;
}

template <class E>
static int win_fwd(const WinDesc& d, hipStream_t st) {
  const long long rows = (long long)d.Sq * d.G, heads = (long long)d.Hk * d.B;
#define GO(DP, NW, NS, OCC) hipLaunchKernelGGL((win_fwd_kernel<E, DP, NW, NS, OCC>), dim3((unsigned)((rows + 32 * NW - 1) / (32 * NW) * heads)), dim3(64 * NW), 0, st, d)
  if (d.D <= 32) GO(32, 4, 3, 4);
  else if (d.D <= 64) GO(64, 4, 3, 3);
  else GO(128, 4, 2, 2);
#undef GO
  return check_launch("window_attention_fwd");
}

size_t window_attention_fwd_workspace_bytes(const WinDesc&) { return 256; }
int window_attention_fwd(const WinDesc& d, int dtype, void* ws, size_t ws_bytes, hipStream_t st) {
  if (int rc = window_attention_check(d, false, "window_attention_fwd")) return rc;
  if (d.B == 0 || d.Sq == 0) return SMBV_OK;
  return dtype == 0 ? win_fwd<ElBf16>(d, st) : win_fwd<ElF16>(d, st);
}

}  // namespace smbv
