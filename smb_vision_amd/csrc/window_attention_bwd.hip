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

template <int DP>
__device__ __forceinline__ void win_stage_keys(unsigned char* img, const uint16_t* base, long long rs, int D, const WinKeys& wk, int u0, int t) {
  constexpr int C = DP / 8;
#pragma unroll
  for (int i = 0; i < 64 * C / 256; i++) {
    const int idx = t + 256 * i, row = idx / C, chunk = idx % C, u = u0 + row;
    u32x4 x = {0, 0, 0, 0};
    if (u < wk.n && chunk * 8 < D) x = *(const u32x4*)(base + (long long)(u < wk.ns ? u : u + wk.jump) * rs + chunk * 8);
    *(u32x4*)(img + win_img<DP>(row, chunk)) = x;
  }
}

template <class E, int DP>
__global__ __launch_bounds__(256, 1) void win_dq_kernel(WinDesc d, const int* __restrict__ expo) {
  constexpr int KS = DP / 16, DT = DP / 32, IMG = 64 * DP * 2;
  using v8 = typename E::v8;
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * IMG];
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
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int x = 0; x < 16; x++) acc[dt][x] = 0.f;
  const int nt = (wk.n + 63) / 64;
  for (int j = 0; j < nt; j++) {
    __syncthreads();
    win_stage_keys<DP>(smem, kb, d.sk.r, d.D, wk, 64 * j, t);
    win_stage_keys<DP>(smem + IMG, vb, d.sv.r, d.D, wk, 64 * j, t);
    __syncthreads();
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
      f32x16 s, dp;
#pragma unroll
      for (int x = 0; x < 16; x++) { s[x] = 0.f; dp[x] = 0.f; }
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        s = E::mfma(__builtin_bit_cast(v8, *(const u32x4*)(smem + win_img<DP>(32 * kt + r31, 2 * ks + h2))), qf[ks], s);
        dp = E::mfma(__builtin_bit_cast(v8, *(const u32x4*)(smem + IMG + win_img<DP>(32 * kt + r31, 2 * ks + h2))), gf[ks], dp);
      }
#pragma unroll
      for (int half = 0; half < 2; half++) {
        v8 ds;
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const int a = 8 * half + x, u = 64 * j + 32 * kt + win_acc_row(a, l), key = u < wk.ns ? u : u + wk.jump;
          const bool vis = u < wk.n && key <= wr.hi && (key >= wr.lo || key < d.sinks);
          ds[x] = (typename E::e)(vis ? fast_exp2(__builtin_fmaf(s[a], c, -lse2)) * (dp[a] - delta) : 0.f);
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) acc[dt] = E::mfma(__builtin_bit_cast(v8, win_read_tr<DP>(smem, 32 * kt + 16 * half, dt, l)), ds, acc[dt]);
      }
    }
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

template <class E, int DP>
__global__ __launch_bounds__(256, 1) void win_dkv_kernel(WinDesc d, const int* __restrict__ expo) {
  constexpr int KS = DP / 16, DT = DP / 32, C = DP / 8, IMG = 64 * DP * 2;
  using v8 = typename E::v8;
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * IMG];
  __shared__ __attribute__((aligned(16))) float st_lse[64], st_delta[64];
  __shared__ int st_lo[64], st_hi[64], st_exp[64];
  const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), r31 = l & 31, h2 = l >> 5;
  int tile, hk, b;
  xcd_block_order((d.Sk + 127) / 128, d.Hk, tile, hk, b);
  const WinSeq seq = win_seq(d, b);
  const int k0 = tile * 128, key = k0 + 32 * w + r31;
  int rlo, rhi;
  win_key_rows(d, seq, k0, k0 + 128, rlo, rhi);
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
  for (int q0 = rlo; q0 < rhi; q0 += 64) {
    __syncthreads();
#pragma unroll
    for (int it = 0; it < 64 * C / 256; it++) {
      const int idx = t + 256 * it, row = idx / C, chunk = idx % C, r = q0 + row;
      u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
      if (r < rhi && chunk * 8 < d.D) {
        const int i = win_div(d, r), head = hk * d.G + (r - i * d.G);
        x = *(const u32x4*)(d.q + b * d.sq.b + i * d.sq.r + head * d.sq.h + chunk * 8);
        y = *(const u32x4*)(d.g + b * d.sg.b + i * d.sg.r + head * d.sg.h + chunk * 8);
      }
      *(u32x4*)(smem + win_img<DP>(row, chunk)) = x;
      *(u32x4*)(smem + IMG + win_img<DP>(row, chunk)) = y;
    }
    if (t < 64) {
      const int r = q0 + t, i = win_div(d, r), head = hk * d.G + (r - i * d.G);
      WinRow wr = win_row(d, seq, i);
      float ls = INFINITY, de = 0.f;
      int ex = WIN_NO_EXP;
      if (r < rhi) {
        const long long at = ((long long)b * d.H + head) * d.Sq + i;
        const float x = d.lse[at];
        if (x != -INFINITY) ls = x * 1.4426950408889634f;
        de = d.delta[at];
        if constexpr (E::half) ex = expo[at];
      } else wr.hi = -1;
      st_lse[t] = ls; st_delta[t] = de; st_lo[t] = wr.lo; st_hi[t] = wr.hi; st_exp[t] = ex;
    }
    __syncthreads();
    float unit = 1.f;
    if constexpr (E::half) {
      int e = st_exp[l];
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
      for (int x = 0; x < 16; x++) { s[x] = 0.f; dp[x] = 0.f; }
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        s = E::mfma(__builtin_bit_cast(v8, *(const u32x4*)(smem + win_img<DP>(32 * qt + r31, 2 * ks + h2))), kf[ks], s);
        dp = E::mfma(__builtin_bit_cast(v8, *(const u32x4*)(smem + IMG + win_img<DP>(32 * qt + r31, 2 * ks + h2))), vf[ks], dp);
      }
#pragma unroll
      for (int half = 0; half < 2; half++) {
        v8 pf, ds;
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const int a = 8 * half + x, row = 32 * qt + win_acc_row(a, l);
          const bool vis = key <= st_hi[row] && (key >= st_lo[row] || key < d.sinks);
          const float p = vis ? fast_exp2(__builtin_fmaf(s[a], c, -st_lse[row])) : 0.f;
          pf[x] = (typename E::e)p;
          float g = vis ? p * (dp[a] - st_delta[row]) : 0.f;
          if constexpr (E::half) g *= unit;
          ds[x] = (typename E::e)g;
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
          dv[dt] = E::mfma(__builtin_bit_cast(v8, win_read_tr<DP>(smem + IMG, 32 * qt + 16 * half, dt, l)), pf, dv[dt]);
          dk[dt] = E::mfma(__builtin_bit_cast(v8, win_read_tr<DP>(smem, 32 * qt + 16 * half, dt, l)), ds, dk[dt]);
        }
      }
    }
  }
  if (key >= d.Sk) return;
  const float f = E::half && emax != WIN_NO_EXP ? ldexpf(d.scale, emax) : d.scale;
  uint16_t* ok = d.dk + b * d.sdk.b + key * d.sdk.r + hk * d.sdk.h;
  uint16_t* ov = d.dv + b * d.sdv.b + key * d.sdv.r + hk * d.sdv.h;
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int rg = 0; rg < 4; rg++) {
      const int d0 = 32 * dt + 8 * rg + 4 * h2;
      if (d0 >= d.D) continue;
      *(u32x2*)(ok + d0) = (u32x2){el_pack<E>(dk[dt][4 * rg] * f, dk[dt][4 * rg + 1] * f), el_pack<E>(dk[dt][4 * rg + 2] * f, dk[dt][4 * rg + 3] * f)};
      *(u32x2*)(ov + d0) = (u32x2){el_pack<E>(dv[dt][4 * rg], dv[dt][4 * rg + 1]), el_pack<E>(dv[dt][4 * rg + 2], dv[dt][4 * rg + 3])};
    }
}

// workspace: delta fp32 [B, H, Sq] | exponents int32 [B, H, Sq] (fp16)
static size_t win_rows_bytes(const WinDesc& d) { return ((size_t)d.B * d.H * d.Sq * 4 + 255) & ~(size_t)255; }
size_t window_attention_bwd_workspace_bytes(const WinDesc& d, int dtype) { return win_rows_bytes(d) * (dtype ? 2 : 1) + 256; }

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
    const dim3 grid((unsigned)((d.Sk + 127) / 128 * d.Hk * d.B));
    if (d.D <= 32) hipLaunchKernelGGL((win_dkv_kernel<E, 32>), grid, dim3(256), 0, st, d, expo);
    else if (d.D <= 64) hipLaunchKernelGGL((win_dkv_kernel<E, 64>), grid, dim3(256), 0, st, d, expo);
    else hipLaunchKernelGGL((win_dkv_kernel<E, 128>), grid, dim3(256), 0, st, d, expo);
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
