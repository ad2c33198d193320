// Windowed attention with sinks: what the forward and the backward share - the operator's description, the geometry of a window and the LDS image.
//
// Query row i of sequence b stands at key position p = i + klen_b - qlen_b (the queries are the LAST rows of their sequence: a training batch has
// qlen = klen, an appended piece or a single token has qlen < klen).  It sees key j iff
//     j < klen_b,   right < 0 or j <= p + right,   left < 0 or j >= p - left or j < sinks.
//     O_i = sum_j P_ij V_j,  P_ij = exp(scale Q_i K_j - LSE_i);  a row that sees nothing has O_i = 0, LSE_i = -inf and gives no gradient.
//
// Heads are grouped: H = G Hk query heads, head h reads key head h / G.  The kernels work on ROWS r = i G + g (query i, head hk G + g): the G heads of a
// group share every key tile that is fetched, and a tile of R rows spans only R / G positions, so its window is narrower.
#pragma once
#include "smbv_common.h"
#include "smbv_kernels.h"

namespace smbv {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(8))) short s16x8;

struct ElBf16 {
  using v8 = bf16x8;
  using e = __bf16;
  static constexpr bool half = false;
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
struct ElF16 {
  using v8 = f16x8;
  using e = _Float16;
  static constexpr bool half = true;
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <class E> __device__ __forceinline__ float el_f(uint16_t u) { return (float)__builtin_bit_cast(typename E::e, u); }
template <class E> __device__ __forceinline__ uint16_t el_u(float f) { return __builtin_bit_cast(uint16_t, (typename E::e)f); }
template <class E> __device__ __forceinline__ unsigned el_pack(float lo, float hi) { return (unsigned)el_u<E>(lo) | ((unsigned)el_u<E>(hi) << 16); }

struct WinStride { long long b, r, h; };  // elements between batches, rows, heads (channels are contiguous)

struct WinDesc {
  int B, Sq, Sk, H, Hk, G, D, left, right, sinks;
  unsigned mG;  // ceil(2^32 / G): r / G by multiplication, exact while r G < 2^32 (checked on the host)
  float scale;
  const int *q_lens, *k_lens;  // per sequence; null = Sq / Sk
  const uint16_t *q, *k, *v, *o_in, *o_lo_in, *g;
  uint16_t *o, *o_lo, *dq, *dk, *dv;
  float* lse;
  WinStride sq, sk, sv, so, sg, sdq, sdk, sdv;
};

struct WinSeq { int klen, qlen, shift; };
__device__ __forceinline__ WinSeq win_seq(const WinDesc& d, int b) {
  WinSeq s;
  s.klen = d.k_lens ? max(0, min(d.k_lens[b], d.Sk)) : d.Sk;
  s.qlen = d.q_lens ? max(0, min(d.q_lens[b], d.Sq)) : d.Sq;
  s.shift = s.klen - s.qlen;
  return s;
}
__device__ __forceinline__ int win_div(const WinDesc& d, int r) { return d.G == 1 ? r : (int)__umulhi((unsigned)r, d.mG); }

// The keys that the queries [i0, i1) can see between them, as ONE run of n: first the ns sinks that lie in front of the window, then the window [lo, hi).
// Sinks therefore cost ns keys of the first tile, not a tile of their own.  Key number of run index u: u < ns ? u : u + jump.
struct WinKeys { int ns, hi, n, jump; };
__device__ __forceinline__ WinKeys win_keys(const WinDesc& d, const WinSeq& s, int i0, int i1) {
  WinKeys w;
  w.hi = d.right < 0 ? s.klen : max(0, min(s.klen, i1 - 1 + s.shift + d.right + 1));
  int lo = d.left < 0 ? 0 : max(0, min(w.hi, i0 + s.shift - d.left));
  w.ns = min(d.sinks, w.hi);
  if (w.ns >= lo) { w.ns = 0; lo = 0; }
  w.n = i1 > i0 ? w.ns + w.hi - lo : 0;
  w.jump = lo - w.ns;
  return w;
}
// What one query sees of the run: indices u with u <= b and (u >= a or u < s); both bounds only grow from query to query.
struct WinView { int a, b, s; };
__device__ __forceinline__ WinView win_view(const WinDesc& d, const WinSeq& q, const WinKeys& w, int i) {
  const int p = i + q.shift, lo = d.left < 0 ? 0 : p - d.left, hi = d.right < 0 ? q.klen - 1 : min(q.klen - 1, p + d.right);
  WinView v;
  v.s = w.ns > 0 ? w.ns : d.sinks;   // (no sinks in front of the window: the run starts at key 0, or there are none)
  v.a = max(w.ns, lo - w.jump);
  v.b = hi >= w.ns + w.jump ? hi - w.jump : min(hi, w.ns - 1);
  return v;
}
// How a tile of T stands to a wave's queries, v0 the first's view and v1 the last's
enum { WIN_NONE = -1, WIN_ALL = 0, WIN_UPPER = 1, WIN_LOWER = 2, WIN_SINKS = 4 };   // nobody sees any of it; all see all; bounds that some row needs, sinks in the tile
template <int T = 64>
__device__ __forceinline__ int win_tile(const WinView& v0, const WinView& v1, int u0) {
  if (u0 > v1.b || (u0 >= v0.s && u0 + T - 1 < v0.a)) return WIN_NONE;
  return (u0 + T - 1 > v0.b ? WIN_UPPER : 0) | (u0 < v1.a && u0 + T - 1 >= v0.s ? WIN_LOWER | (u0 < v0.s ? WIN_SINKS : 0) : 0);
}
// Masks 32 scores: accumulator row 0 of this lane is run index o (a tile's edge needs one bound, and each costs two instructions a score)
__device__ __forceinline__ void win_mask(f32x16& s, int kind, const WinView& v, int o) {
  if (kind & WIN_UPPER) {
    const int b = v.b - o;
#pragma unroll
    for (int x = 0; x < 16; x++) s[x] = (x & 3) + 8 * (x >> 2) <= b ? s[x] : -INFINITY;
  }
  if (kind & WIN_LOWER) {
    const int a = v.a - o;
    if (kind & WIN_SINKS) {
      const int n = v.s - o;
#pragma unroll
      for (int x = 0; x < 16; x++) s[x] = (x & 3) + 8 * (x >> 2) >= a || (x & 3) + 8 * (x >> 2) < n ? s[x] : -INFINITY;
    } else {
#pragma unroll
      for (int x = 0; x < 16; x++) s[x] = (x & 3) + 8 * (x >> 2) >= a ? s[x] : -INFINITY;
    }
  }
}

// LDS image of a tile: rows of DP 16-bit elements (C = DP / 8 chunks of 16 bytes), chunk c of row r at chunk c ^ f(r).  f serves both ways in which a
// tile feeds the matrix pipe: 16 consecutive rows of one chunk (ds_read_b128) fall on 16 different chunks of 256 bytes, and the 4 rows x 64 bytes of a
// transposed read (ds_read_b64_tr_b16) on different 64-byte groups.
template <int DP> __device__ __forceinline__ int win_img(int row, int chunk) {
  if constexpr (DP == 128) return row * 256 + ((chunk ^ (((row & 3) << 2) | ((row >> 2) & 3))) << 4);
  else if constexpr (DP == 64) return row * 128 + ((chunk ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3))) << 4);
  else return row * 64 + ((chunk ^ ((row >> 2) & 3)) << 4);
}

// LDS addresses of this lane's operands in a tile at address `base`; everything else - the tile's slot, the 32 or 16 rows inside it - is an immediate.
//   row[ks]    16 bytes of row (lane & 31): the A or B operand of a product over the channels
//   tr[dt][e]  transposed: the A operand (32 channels x 16 rows) of a product over the rows; its 16 rows are 8 e + 4 (lane >> 5) + 0..3, e = 0, 1, which is
//              the order in which an accumulator's registers hold them: exponentiated scores are the B operand as they are
// (f has period 16 in the row, so steps of 16 rows leave the chunk's place alone)
template <int DP> struct WinRead {
  static constexpr int KS = DP / 16, DT = DP / 32;
  unsigned row[KS], tr[DT][2];
  __device__ __forceinline__ WinRead(unsigned base, int l) {
    const int g1 = (l >> 4) & 1, qq = (l >> 2) & 3, pp = l & 3, h2 = l >> 5;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) row[ks] = base + win_img<DP>(l & 31, 2 * ks + h2);
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int e = 0; e < 2; e++) tr[dt][e] = base + win_img<DP>(8 * e + 4 * h2 + qq, 4 * dt + 2 * g1 + (pp >> 1)) + ((pp & 1) << 3);
  }
  __device__ __forceinline__ u32x4 rows(int ks, int off) const { return *(const __attribute__((address_space(3))) u32x4*)(row[ks] + off); }
  __device__ __forceinline__ s16x8 cols(int dt, int off) const {
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(tr[dt][0] + off));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(tr[dt][1] + off));
    return (s16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  // (an LDS instruction's immediate reaches 64 KiB: a ring of 128 KiB is read from one half, then the other)
  __device__ __forceinline__ void move(int by) {
#pragma unroll
    for (int ks = 0; ks < KS; ks++) { row[ks] += by; asm volatile("" : "+v"(row[ks])); }   // (or it is added at every read)
#pragma unroll
    for (int dt = 0; dt < DT; dt++) { tr[dt][0] += by; tr[dt][1] += by; asm volatile("" : "+v"(tr[dt][0]), "+v"(tr[dt][1])); }
  }
};
__device__ __forceinline__ void win_drain() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }  // (no copy may outlive its workgroup)
// Walk n tiles of a ring of NS slots of SLOT bytes: arrive(), stage(tile, slot), use(tile, offset of its slot from the reader's addresses)
template <int NS, int SLOT, class Arrive, class Stage, class Use, class Move>
__device__ __forceinline__ void win_walk(int n, Arrive arrive, Stage stage, Use use, Move move) {
  constexpr int HALF = NS * SLOT <= 65536 ? NS : 65536 / SLOT;   // slots within reach of one address
  static_assert(NS % HALF == 0 && NS / HALF <= 2, "one or two halves");
#pragma unroll
  for (int s = 0; s < NS - 1; s++) stage(s, s);
  for (int j = 0; j < n; j += NS) {
#pragma unroll
    for (int s = 0; s < NS; s++) {
      if (j + s >= n) break;
      arrive();
      stage(j + s + NS - 1, (s + NS - 1) % NS);
      use(j + s, (s % HALF) * SLOT);
      if constexpr (HALF < NS) {
        if (s % HALF == HALF - 1) move(s < HALF ? HALF * SLOT : -HALF * SLOT);
      }
    }
  }
  win_drain();
}

// Workgroups of one key head share its keys and queries, and an XCD (every eighth workgroup) has an L2 of its own: whole key heads go to one XCD, eight at a
// time, and what is left of them is dealt out in eight contiguous runs.  (Contiguous runs for everything put the long sequences of a ragged batch on a few XCDs.)
__device__ __forceinline__ void win_block_order(int nt, int Hk, int B, int& tile, int& hk, int& b) {
  const int id = blockIdx.x, heads = Hk * B, whole = heads >> 3, xcd = id & 7, slot = id >> 3;
  int hb;
  if (slot < whole * nt) {
    hb = (slot / nt) * 8 + xcd;
    tile = slot % nt;
  } else {
    const int n = (heads & 7) * nt, s = slot - whole * nt, q8 = n >> 3, r8 = n & 7;
    const int g = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + s;
    hb = whole * 8 + g / nt;
    tile = g % nt;
  }
  hk = hb % Hk;
  b = hb / Hk;
}

// ---- tiles of 64 rows, copied global -> LDS without passing registers ----------------------------------------------------------------------------------
// The copy is issued from asm, where the compiler does not see it (it would wait for every copy in flight in front of every LDS read).  A ring of NS slots: at
// tile j the kernels wait with win_arrived() for tile j, not for the NS - 2 tiles behind it, and issue the copy of tile j + NS - 1 into the slot that tile
// j - 1 has left.  The count is the same for every tile (one past the end copies rows that are there anyway).
// One wave-instruction moves 1 KiB: lane i's 16 bytes go to LDS address lds + 16 i, from a uniform base + 32-bit offset or from a 64-bit address of its own.
__device__ __forceinline__ void win_dma_off(const void* sbase, unsigned voff, unsigned lds) {
  unsigned keep;
  asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "s"(lds), "v"(voff), "s"(sbase) : "memory");
}
__device__ __forceinline__ void win_dma_ptr(const void* p, unsigned lds) {
  unsigned keep;
  asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "s"(lds), "v"(p) : "memory");
}
__device__ __forceinline__ void win_dma4_ptr(const void* p, unsigned lds) {   // 4 bytes a lane
  unsigned keep;
  asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %2, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "s"(lds), "v"(p) : "memory");
}
// This wave's copies have landed but for the youngest N, its reads of the slot that is filled next have returned, and so say all waves.
template <int N>
__device__ __forceinline__ void win_arrived() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// a pointer that is the same in every lane, in scalar registers
__device__ __forceinline__ const uint16_t* win_uniform(const uint16_t* p) {
  const unsigned long long a = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((int)(unsigned)a), hi = __builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32));
  return (const uint16_t*)(((unsigned long long)hi << 32) | lo);
}

// What one of NW waves copies of a tile: piece p is the rows (NP w + p) R .. + R - 1.  The image's chunk permutation is applied on the source side.  A chunk
// past the head's width takes the last one: the other operand of its products is zero there, or their result is not stored.
template <int DP, int NW>
struct WinCopy {
  static constexpr int C = DP / 8, NP = DP / 8 / NW, R = 64 / C;
  static_assert(NP >= 1, "a wave copies whole pieces");
  int row[NP], chunk[NP];
  __device__ __forceinline__ WinCopy(int w, int l, int D) {
#pragma unroll
    for (int p = 0; p < NP; p++) {
      row[p] = (w * NP + p) * R + l / C;
      chunk[p] = min((win_img<DP>(row[p], l % C) - row[p] * DP * 2) >> 4, D / 8 - 1);
    }
  }
  // byte offsets of rows that lie at a fixed distance
  __device__ __forceinline__ void offsets(unsigned (&off)[NP], long long rs) const {
#pragma unroll
    for (int p = 0; p < NP; p++) off[p] = (unsigned)(row[p] * (unsigned)rs * 2 + chunk[p] * 16);
  }
  // tile of run indices u0 .. u0 + 63 of the keys (an index past the run takes the run's last key: it is masked)
  __device__ __forceinline__ void keys(const uint16_t* base, long long rs, const unsigned (&off)[NP], const WinKeys& wk, int u0, unsigned lds) const {
    if (u0 + 64 <= wk.n && (u0 >= wk.ns || u0 + 64 <= wk.ns)) {
      const uint16_t* s = win_uniform(base + (long long)(u0 < wk.ns ? u0 : u0 + wk.jump) * rs);
#pragma unroll
      for (int p = 0; p < NP; p++) win_dma_off(s, off[p], lds + p * 1024);
    } else {
#pragma unroll
      for (int p = 0; p < NP; p++) {
        const int u = min(u0 + row[p], wk.n - 1);
        win_dma_ptr(base + (long long)(u < wk.ns ? u : u + wk.jump) * rs + chunk[p] * 8, lds + p * 1024);
      }
    }
  }
};

// Left alone the compiler puts an LDS read right in front of the product that waits for it.  Code on the two sides of this line stays there: operands are read
// on one side and used on the other, where the next ones are read.
#define WIN_AHEAD() __builtin_amdgcn_sched_barrier(0)
// The basic block's products and vector instructions in turn: N times one and V
template <int N, int V> __device__ __forceinline__ void win_weave() {
#pragma unroll
  for (int i = 0; i < N; i++) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
  }
}

// x of this lane and of lane l ^ 32
__device__ __forceinline__ void win_halves(float x, float& u, float& v) {
  typedef unsigned u32x2v __attribute__((ext_vector_type(2)));
  const unsigned a = __builtin_bit_cast(unsigned, x);
  const u32x2v sw = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  unsigned lo = sw[0], hi = sw[1];
  asm volatile("" : "+v"(lo), "+v"(hi));  // (kept apart: hipcc folds an operation on the two results of one swap)
  u = __builtin_bit_cast(float, lo);
  v = __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float win_halves_max(float x) { float u, v; win_halves(x, u, v); return fmaxf(u, v); }
__device__ __forceinline__ float win_halves_sum(float x) { float u, v; win_halves(x, u, v); return u + v; }

int window_attention_check(const WinDesc& d, bool backward, const char* what, bool sizes_only = false);
size_t window_attention_fwd_workspace_bytes(const WinDesc& d);
int window_attention_fwd(const WinDesc& d, int dtype, void* ws, size_t ws_bytes, hipStream_t st);
size_t window_attention_bwd_workspace_bytes(const WinDesc& d, int dtype);
int window_attention_bwd(const WinDesc& d, int dtype, void* ws, size_t ws_bytes, hipStream_t st);
}  // namespace smbv
