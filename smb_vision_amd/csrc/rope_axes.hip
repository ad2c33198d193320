// Rotary positions with several axes (time, height, width, ...) on queries and keys, and the transposed map for their gradients.
//
// Pair p of a head's first 2 P channels belongs to axis a(p) (the axes own consecutive runs of pairs) and turns by  angle = pos[a(p)][b, s] * inv_freq[p]:
//     (y0, y1) = (x0 cos - x1 sin, x0 sin + x1 cos),   transposed: the angle's sign flips;   channels from 2 P on are copied.
// Pairs are (p, p + P) or, interleaved, (2 p, 2 p + 1).
// Bound by HBM: every element is read and written once (20,480 tokens, 12 heads on 12 of 64 channels in bf16, 126 MB: 24.8 us, 5.1 TB/s).  A workgroup forms the cosines and sines of its tokens once in LDS and streams all heads of
// these tokens past them.  The angle is formed and reduced to one turn in 64 bits: position * frequency in 32 bits is off by 2^-24 of the whole angle, which
// at position 100,000 is 0.006 rad.
#include "smbv_common.h"
#include "smbv_kernels.h"

namespace smbv {

template <class T> struct RopeIo;
template <> struct RopeIo<float> {
  static __device__ __forceinline__ float ld(float x) { return x; }
  static __device__ __forceinline__ float st(float x) { return x; }
};
template <> struct RopeIo<__bf16> {
  static __device__ __forceinline__ float ld(__bf16 x) { return (float)x; }
  static __device__ __forceinline__ __bf16 st(float x) { return (__bf16)x; }
};
template <> struct RopeIo<_Float16> {
  static __device__ __forceinline__ float ld(_Float16 x) { return (float)x; }
  // (kept apart from the sum in front of it: v_fma_mixlo_f16 rounds the two at once, and some of a variant's elements would have it and others not)
  static __device__ __forceinline__ _Float16 st(float x) { asm("" : "+v"(x)); return (_Float16)x; }
};
template <class T, int V> struct __attribute__((aligned(V > 2 ? sizeof(T) * V : sizeof(T)))) RopeVec { T e[V]; };  // (V = 2: the fallback for any alignment)

static constexpr int ROPE_LDS_PAIRS = 2048;  // angles of one workgroup's tokens: 16 KB

// (the contraction is spelled out: every alignment's variant rounds alike)
// V elements to an access: V pairs of halves, V / 2 interleaved pairs (V = 1: one pair of halves; V = 2 with ILV: one interleaved pair)
template <class T, int V, bool ILV>
__global__ __launch_bounds__(256) void rope_axes_kernel(RopeAxesDesc d, int tokens_per_block) {
  __shared__ float2 cs[ROPE_LDS_PAIRS];
  const int t = threadIdx.x;
  const long long n = (long long)d.B * d.S, tok0 = (long long)blockIdx.x * tokens_per_block;
  const int nt = (int)(n - tok0 < tokens_per_block ? n - tok0 : tokens_per_block);
  for (int x = t; x < nt * d.P; x += 256) {
    const int tk = x / d.P, p = x - tk * d.P;
    const long long tok = tok0 + tk;
    const int b = (int)(tok / d.S), s = (int)(tok - (long long)b * d.S);
    const int a = (p >= d.end[0]) + (p >= d.end[1]) + (p >= d.end[2]);
    const long long at = a * d.pos_a + b * d.pos_b + s * d.pos_s;
    const double pos = d.pos64 ? (double)((const long long*)d.pos)[at] : (double)((const int*)d.pos)[at];
    const double turns = pos * (double)d.inv_freq[p] * 0.15915494309189533577;
    const float f = (float)(turns - rint(turns));   // in [-1/2, 1/2]
    float sn, c;
    sincospif(2.f * f, &sn, &c);
    cs[x] = make_float2(c, d.transpose ? -sn : sn);
  }
  __syncthreads();
  const int ng = ILV ? 2 * d.P / V : d.P / V;                                   // groups of pairs of a head
  const int gap = d.D - 2 * d.P, nc = gap / V, per_head = ng + (d.copy ? nc : 0);  // ... and groups of copied channels
  const int per_tok = per_head * (d.H + d.Hk);
  for (int x = t; x < nt * per_tok; x += 256) {
    const int tk = x / per_tok, y = x - tk * per_tok, h = y / per_head, g = y - h * per_head;
    const long long tok = tok0 + tk;
    const int b = (int)(tok / d.S), s = (int)(tok - (long long)b * d.S);
    const bool isq = h < d.H;
    const int hh = isq ? h : h - d.H;
    const T* in = (const T*)(isq ? d.q : d.k) + (isq ? b * d.sq[0] + s * d.sq[1] + hh * d.sq[2] : b * d.sk[0] + s * d.sk[1] + hh * d.sk[2]);
    T* out = (T*)(isq ? d.qo : d.ko) + (isq ? b * d.sqo[0] + s * d.sqo[1] + hh * d.sqo[2] : b * d.sko[0] + s * d.sko[1] + hh * d.sko[2]);
    const float2* a = cs + tk * d.P;
    using VT = RopeVec<T, V>;
    if (g >= ng) {
      const int at = 2 * d.P + (g - ng) * V;
      *(VT*)(out + at) = *(const VT*)(in + at);
    } else if constexpr (ILV) {
      VT v = *(const VT*)(in + g * V);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 w = a[(g * V + e) >> 1];
        const float x0 = RopeIo<T>::ld(v.e[e]), x1 = RopeIo<T>::ld(v.e[e + 1]);
        v.e[e] = RopeIo<T>::st(__builtin_fmaf(x0, w.x, -(x1 * w.y)));
        v.e[e + 1] = RopeIo<T>::st(__builtin_fmaf(x0, w.y, x1 * w.x));
      }
      *(VT*)(out + g * V) = v;
    } else {
      VT v0 = *(const VT*)(in + g * V), v1 = *(const VT*)(in + d.P + g * V);
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float2 w = a[g * V + e];
        const float x0 = RopeIo<T>::ld(v0.e[e]), x1 = RopeIo<T>::ld(v1.e[e]);
        v0.e[e] = RopeIo<T>::st(__builtin_fmaf(x0, w.x, -(x1 * w.y)));
        v1.e[e] = RopeIo<T>::st(__builtin_fmaf(x0, w.y, x1 * w.x));
      }
      *(VT*)(out + g * V) = v0;
      *(VT*)(out + d.P + g * V) = v1;
    }
  }
}

template <class T>
static int rope_axes_t(const RopeAxesDesc& d, hipStream_t st) {
  constexpr int W = 16 / sizeof(T);
  const long long n = (long long)d.B * d.S;
  // enough blocks to fill the chip, at most ROPE_LDS_PAIRS angles a block
  const int tpb = (int)std::max<long long>(1, std::min<long long>(ROPE_LDS_PAIRS / d.P, n / 2048));
  if (n / tpb >= (1 << 24) - 1) { set_error("rope_axes: %d x %d tokens are too many for one call", d.B, d.S); return SMBV_ERR_SHAPE; }   // (a launch ends at 2^32 threads)
  const dim3 grid((unsigned)((n + tpb - 1) / tpb)), blk(256);
  long long bits = (d.H ? ((uintptr_t)d.q | (uintptr_t)d.qo) / sizeof(T) | d.sq[0] | d.sq[1] | d.sq[2] | d.sqo[0] | d.sqo[1] | d.sqo[2] : 0) |
                   (d.Hk ? ((uintptr_t)d.k | (uintptr_t)d.ko) / sizeof(T) | d.sk[0] | d.sk[1] | d.sk[2] | d.sko[0] | d.sko[1] | d.sko[2] : 0) |
                   (d.interleaved ? 2 * d.P : d.P) | d.D;
  const bool wide = (bits & (W - 1)) == 0;
  if (d.interleaved) {
    if (wide) hipLaunchKernelGGL((rope_axes_kernel<T, W, true>), grid, blk, 0, st, d, tpb);
    else hipLaunchKernelGGL((rope_axes_kernel<T, 2, true>), grid, blk, 0, st, d, tpb);
  } else {
    if (wide) hipLaunchKernelGGL((rope_axes_kernel<T, W, false>), grid, blk, 0, st, d, tpb);
    else hipLaunchKernelGGL((rope_axes_kernel<T, 1, false>), grid, blk, 0, st, d, tpb);
  }
  return check_launch("rope_axes");
}

int rope_axes(const RopeAxesDesc& d, int dtype, hipStream_t st) {
  if (d.B < 0 || d.S < 0 || d.H < 0 || d.Hk < 0) { set_error("rope_axes: bad shape B=%d S=%d H=%d Hk=%d", d.B, d.S, d.H, d.Hk); return SMBV_ERR_SHAPE; }
  if (d.D <= 0 || (d.D & 1) || d.D > 1024 || d.P <= 0 || d.P > d.D / 2) { set_error("rope_axes: head width %d (even, up to 1024) with %d rotated pairs", d.D, d.P); return SMBV_ERR_SHAPE; }
  if (d.B == 0 || d.S == 0 || d.H + d.Hk == 0) return SMBV_OK;
  if ((long long)d.B * d.S >= (1ll << 31) || (long long)(d.H + d.Hk) * d.D >= (1 << 19)) { set_error("rope_axes: %d x %d tokens of %d heads are too many for one call", d.B, d.S, d.H + d.Hk); return SMBV_ERR_SHAPE; }
  if ((d.H && (!d.q || !d.qo)) || (d.Hk && (!d.k || !d.ko)) || !d.pos || !d.inv_freq) { set_error("rope_axes: null operand"); return SMBV_ERR_ARG; }
  const unsigned am = dtype == 2 ? 3 : 1;
  if (((uintptr_t)d.q | (uintptr_t)d.k | (uintptr_t)d.qo | (uintptr_t)d.ko) & am) { set_error("rope_axes: alignment"); return SMBV_ERR_ALIGN; }
  return dtype == 0 ? rope_axes_t<__bf16>(d, st) : dtype == 1 ? rope_axes_t<_Float16>(d, st) : rope_axes_t<float>(d, st);
}

}  // namespace smbv
