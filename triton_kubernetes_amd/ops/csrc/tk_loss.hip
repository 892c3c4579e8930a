// Losses of a language model's output head on MI355X (gfx950): the logits z = X W^T of N tokens
// over a vocabulary of V are never stored.
//
// Both losses compare the softmax q of a row's logits (at a temperature T) with K sparse
// targets (id_k, p_k), sum_k p_k = 1:
//
//     lse  = log sum_v exp(z_v / T)
//     loss = T^2 sum_k p_k (log p_k - z_{id_k} / T + lse)
//     dloss/dz_v = T (q_v - sum_{k: id_k = v} p_k)
//
// Cross entropy is K = 1, p = 1, T = 1; distillation takes p from a teacher's top logits.
//
// Forward: one matrix product whose epilogue reduces every tile of 256 vocabulary entries to
// a running maximum and sum per token (k_logits<LSE>), a dot product per target (k_dots), and
// a join over the tiles (k_loss).
// Backward, in pieces of the vocabulary: the logits of the piece are computed again, and the
// epilogue turns them into their 16-bit derivative dl (k_logits<DL>; the sparse targets are
// put in by k_fix); then dX += dl W and dW = dl^T X, two matrix products that read dl while
// the last-level cache still holds it.
//
// Rows without a target (masked tokens) are left out before any product: k_gather packs the
// others into Xc, so that whatever the masked rows hold (infinities, NaN) reaches nothing and
// costs nothing.  The number of packed rows stays on the device; the tiles beyond it end at once.
//
// C ABI for ctypes: triton_kubernetes_amd/ops/loss.py.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <mutex>

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;

static thread_local char g_err[512];

extern "C" const char* tkl_last_error() { return g_err; }

static int set_err(const char* what, hipError_t e) {
  snprintf(g_err, sizeof(g_err), "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
  return (int)e == 0 ? -1 : (int)e;
}

// One call's tensors and sizes (ops/loss.py:_Args holds the same fields in the same order).
struct tkl_args {
  long long n, d, v, k;        // tokens, width, vocabulary, targets per token
  long long ldx, ldw, ldg;     // row strides of x and w, stride of the upstream gradient (elements)
  long long ignore;            // cross entropy: the target that means "no loss"
  long long piece, splits;     // backward: vocabulary entries per piece, splits of the dX product
  int dev, f16, distill, reduction;  // reduction 0 none, 1 sum, 2 mean
  float temperature;
  int want;                    // backward: 1 dX, 2 dW, 3 both
  const void *x, *w, *ids, *teacher, *grad;
  void *loss, *xc, *lse, *zk, *p, *rowloss, *rowmap, *posof, *count;  // kept from forward to backward
  void *flag;                  // distillation: whether a row has a target
  void *part;                  // forward: tile maxima and sums
  void *wc;                    // a padded copy of w, where w's rows are not 16-byte aligned
  void *dl, *dxpart, *factor;  // backward workspaces
  void *dx, *dw;
  void* stream;
};

namespace {

constexpr int THREADS = 512;  // of the matrix products: 8 waves, one 256x256 tile
constexpr int TILE = 256;
constexpr int KT = 64;  // K elements of a step (128 bytes of a row)
constexpr int HBYTES = 128 * KT * 2;
constexpr int LDS = 8 * HBYTES;
constexpr unsigned FAR = 0x40000000u;  // an offset past every descriptor's end: the copy writes zeros
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

template <bool F16>
struct Type;
template <>
struct Type<false> {
  using T = __bf16;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
};
template <>
struct Type<true> {
  using T = _Float16;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
};

template <typename T>
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
  typedef __attribute__((ext_vector_type(2))) T t2;
  const t2 v = {(T)lo, (T)hi};
  return __builtin_bit_cast(unsigned, v);
}

// Block -> tile, XCD-aware: workgroups go round-robin over the 8 XCDs, so XCD x takes the
// x-th run of tiles and the tiles of a run share panels in that XCD's L2.
__device__ __forceinline__ void tile_of(int b, int nwg, int tiles_m, int tiles_n, int* tm, int* tn) {
  const int xcd = b & 7, q = nwg >> 3, rem = nwg & 7;
  const int w = (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + (b >> 3);
  constexpr int GROUP_M = 8;
  const int per_group = GROUP_M * tiles_n;
  const int g = w / per_group, first_m = g * GROUP_M;
  const int rows = min(tiles_m - first_m, GROUP_M);
  const int in = w - g * per_group;
  *tm = first_m + in % rows;
  *tn = in / rows;
}

__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");  // the barrier alone does not hold the compiler's LDS reads back
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// 16 bytes a lane from a buffer (offset `voff`, zeros past its end) to LDS at `lds` + 16 lane.
// In asm, because the compiler would wait for every copy in flight before each
// ds_read_b64_tr_b16 (2.25 instead of 1.83 ms for k_dx and k_dw at 8192 x 4096 x 32768); product() does the
// waiting.  The copy has no register output; it reads its operands when it is issued.
__device__ __forceinline__ void copy16(u32x4 buffer, unsigned voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff),
               "s"(buffer)
               : "memory", "m0");
}
__device__ __forceinline__ u32x4 buffer_of(const char* base, unsigned bytes) {
  const unsigned long long b = reinterpret_cast<unsigned long long>(base);
  // (the readfirstlanes are no instructions where the values are scalar already: they only
  // make the compiler keep the descriptor in scalar registers)
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)b), hi = __builtin_amdgcn_readfirstlane((unsigned)(b >> 32));
  return u32x4{lo, hi & 0xffffu, (unsigned)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}

// One 256-wide panel of an operand.  ALONG: a row of the panel lies along K (128 rows of 128
// bytes are a half-tile); else K is the matrix's row index (64 rows of 128 columns), and the
// fragments are transposed on their way out of LDS.
template <bool ALONG>
struct Panel;

// Rows along K: LDS image [128 rows][8 chunks of 16 bytes], chunk c of row r at c ^ (r/2 & 7)
// (the 16 rows of a fragment read land in 16 bank slots).
template <>
struct Panel<true> {
  const char* base;
  unsigned ld, kbytes;  // row stride, valid bytes of a row
  unsigned bytes;       // from base to the end of the last valid row (at most 256 rows: below 2^31)
  unsigned voff, chunk;

  __device__ __forceinline__ Panel(const void* m, long long ldb, int row0, int rows, int k0, int k, int tid) {
    base = static_cast<const char*>(m) + (long long)row0 * ldb + (long long)k0 * 2;
    ld = (unsigned)ldb;
    kbytes = k * 2;
    bytes = (min(rows - row0, TILE) - 1) * ld + kbytes;
    const int r = tid >> 3;
    chunk = ((tid & 7) ^ ((r >> 1) & 7)) * 16;
    voff = r * ld + chunk;
  }
  // the two copies of a thread for half-tile h of step t, to LDS at dst (of this wave)
  __device__ __forceinline__ void stage(int t, int h, unsigned dst) const {
    const unsigned k = t * (KT * 2), v = k + chunk < kbytes ? voff : FAR;  // past the row's end: zeros
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned at = (h * 128 + i * 64) * ld + k;
      copy16(buffer_of(base + at, bytes > at ? bytes - at : 0), v, dst + i * THREADS * 16);
    }
  }
  // the 16 rows at r0 of a half-tile, K chunk kk of 32
  __device__ __forceinline__ static u32x4 frag(const char* img, int r0, int kk, int lane) {
    const int r = r0 + (lane & 15), c = kk * 4 + (lane >> 4);
    return *reinterpret_cast<const u32x4*>(img + r * 128 + ((c ^ ((r >> 1) & 7)) * 16));
  }
};

// K down the rows: LDS image [64 k][8 units of 32 bytes], unit u of row k at u ^ f(k), f(k) =
// (k & 3) | (k >> 3 & 1) << 2: the 8 rows that half a wave reads at once land on different
// banks.  ds_read_b64_tr_b16 gives lane c of a 16-lane group the 4 values of column c from the
// 4 rows that the group reads.
template <>
struct Panel<false> {
  const char* base;
  int krows;
  unsigned ld, width;  // row stride, valid bytes of a row from base on
  unsigned voff;

  __device__ __forceinline__ Panel(const void* m, long long ldb, int col0, int cols, int k0, int k, int tid) {
    base = static_cast<const char*>(m) + (long long)k0 * ldb + (long long)col0 * 2;
    ld = (unsigned)ldb;
    krows = k;
    width = (cols - col0) * 2;
    const int r = tid >> 4, c = tid & 15;
    const int f = (r & 3) | ((r >> 1) & 4);
    voff = r * ld + ((((c >> 1) ^ f) << 1) | (c & 1)) * 16;
  }
  __device__ __forceinline__ void stage(int t, int h, unsigned dst) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k = t * KT + i * 32, rows = min(krows - k, 32);
      const unsigned end = rows > 0 ? (rows - 1) * ld + width : 0;  // 32 rows of at most 2^25 bytes
      copy16(buffer_of(base + (unsigned long long)(unsigned)k * ld + h * 256, end > h * 256u ? end - h * 256u : 0), voff,
             dst + i * THREADS * 16);
    }
  }
  __device__ __forceinline__ static u32x4 frag(const char* img, int c0, int kk, int lane) {
    const int q = lane >> 4, l = lane & 15;
    const int f = (l >> 2) | ((q & 1) << 2);
    const char* p = img + (kk * 32 + q * 8 + (l >> 2)) * 256 + (((c0 >> 4) ^ f) * 32) + (l & 3) * 8;
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * 256)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
};

typedef f32x4 Acc[2][2][4][2];  // [mh][nh][i][j]

// One 256x256 tile of A B^T over nk steps of 64.  Element (mh, nh, i, j, e) of a lane is
// row mh*128 + wr*64 + i*16 + (lane/16)*4 + e and column nh*128 + wc*32 + j*16 + lane%16.
//
// The schedule is the one of tk_gemm_screen.hip's k_gemm8: LDS holds half-tiles of two steps,
// a step is two phases of 32 matrix instructions per wave, and the wave groups wr = 0 and 1
// run one barrier apart, so that on every SIMD one wave feeds the matrix pipe while the other
// reads LDS and issues copies.
template <bool F16, bool AA, bool BA>
__device__ __forceinline__ void product(Acc& acc, char* smem, const Panel<AA>& pa, const Panel<BA>& pb, int nk,
                                        int tid) {
  const int lane = tid & 63, wid = tid >> 6, wr = wid >> 2, wc = wid & 3;
#pragma unroll
  for (int mh = 0; mh < 2; ++mh)
#pragma unroll
    for (int nh = 0; nh < 2; ++nh)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[mh][nh][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (nk <= 0) return;

  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)smem +
                        __builtin_amdgcn_readfirstlane(wid) * 64 * 16;
  auto slot = [&](int t, int h) { return smem + ((t & 1) * 4 + h) * HBYTES; };
  auto stage = [&](int t, int h) {  // h: 0 A0, 1 A1, 2 B0, 3 B1
    const unsigned dst = lds0 + ((t & 1) * 4 + h) * HBYTES;
    if (h < 2) pa.stage(t, h, dst);
    else pb.stage(t, h - 2, dst);
  };
  u32x4 a[4][2], b[2][2][2];
  auto read_a = [&](int t, int mh) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) a[i][kk] = Panel<AA>::frag(slot(t, mh), wr * 64 + i * 16, kk, lane);
  };
  auto read_b = [&](int t, int nh) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) b[nh][j][kk] = Panel<BA>::frag(slot(t, 2 + nh), wc * 32 + j * 16, kk, lane);
  };
  auto quad = [&](int mh, int nh) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
          acc[mh][nh][i][j] = Type<F16>::mfma(a[i][kk], b[nh][j][kk], acc[mh][nh][i][j]);
    __builtin_amdgcn_s_setprio(0);
  };
  // keep every matrix instruction between its phase's two barriers
  auto pin_frags = [&](bool with_b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(a[i][0]), "+v"(a[i][1]));
    if (with_b) {
#pragma unroll
      for (int nh = 0; nh < 2; ++nh)
#pragma unroll
        for (int j = 0; j < 2; ++j) asm volatile("" : "+v"(b[nh][j][0]), "+v"(b[nh][j][1]));
    }
  };
  auto pin_acc = [&](int mh) {
#pragma unroll
    for (int nh = 0; nh < 2; ++nh)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) asm volatile("" : "+v"(acc[mh][nh][i][j]));
  };

  stage(0, 0);
  stage(0, 2);
  stage(0, 3);
  stage(0, 1);
  if (nk > 1) {
    stage(1, 0);
    stage(1, 2);
    asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  barrier();
  if (wr == 1) barrier();  // the stagger
  for (int t = 0; t < nk; ++t) {
    const bool more1 = t + 1 < nk, more2 = t + 2 < nk;
    read_a(t, 0);
    read_b(t, 0);
    __builtin_amdgcn_sched_barrier(0);  // B1's reads last: the wait below leaves only them
    read_b(t, 1);
    if (more1) {
      stage(t + 1, 3);
      stage(t + 1, 1);
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    if constexpr (BA) asm volatile("s_waitcnt lgkmcnt(4)" ::: "memory");
    else asm volatile("s_waitcnt lgkmcnt(8)" ::: "memory");
    barrier();
    pin_frags(true);
    quad(0, 0);
    quad(0, 1);
    pin_acc(0);
    barrier();
    read_a(t, 1);
    if (more2) {
      stage(t + 2, 0);
      stage(t + 2, 2);
      asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    }
    barrier();
    pin_frags(false);
    quad(1, 1);
    quad(1, 0);
    pin_acc(1);
    barrier();
  }
  if (wr == 0) barrier();  // the other group's extra barrier
}

struct Lane {
  int lane, wr, wc, fr, fq;
  __device__ __forceinline__ Lane(int tid) {
    lane = tid & 63;
    wr = tid >> 8;
    wc = (tid >> 6) & 3;
    fr = lane & 15;
    fq = lane >> 4;
  }
};

// (m, s) of a softmax: maximum and sum of exp2(. - m).  An empty side has m = -inf, s = 0.
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float a = m == top ? 1.f : exp2f(m - top), b = m2 == top ? 1.f : exp2f(m2 - top);
  s = s * a + s2 * b;
  m = top;
}

// z^T of 256 vocabulary entries (A = W) by 256 tokens (B = Xc), so that a lane holds 32
// entries of each of 4 tokens and the softmax's sums need two shuffles a token.
// LSE: writes part[2 * tile + wr][token] = (max, sum).  DL: writes f (q - 0) in 16 bits.
// sc = log2(e) / T.
template <bool F16, bool DL>
__global__ __launch_bounds__(THREADS) void k_logits(const void* __restrict__ w, long long ldw,
                                                    const void* __restrict__ xc, long long ldxc, int v0, int vend,
                                                    int d, const int* __restrict__ count, int n, float sc,
                                                    float2* __restrict__ part, const float* __restrict__ lse,
                                                    const float* __restrict__ factor, void* __restrict__ dl,
                                                    long long lddl) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using T = typename Type<F16>::T;
  const int rows = count[0];
  const int tiles_v = (vend - v0 + TILE - 1) / TILE, tiles_n = (rows + TILE - 1) / TILE;
  const int nwg = tiles_v * tiles_n;
  if ((int)blockIdx.x >= nwg) return;
  int tv, tn;
  tile_of(blockIdx.x, nwg, tiles_v, tiles_n, &tv, &tn);
  const int tid = threadIdx.x;
  const Panel<true> pa(w, ldw, v0 + tv * TILE, vend, 0, d, tid), pb(xc, ldxc, tn * TILE, rows, 0, d, tid);
  Acc acc;
  product<F16, true, true>(acc, smem, pa, pb, (d + KT - 1) / KT, tid);

  const Lane l(tid);
  const int vb = tv * TILE + l.wr * 64 + l.fq * 4;  // the lane's first entry, in the piece
  const int vn = vend - v0;
  const bool whole = (tv + 1) * TILE <= vn;
#pragma unroll
  for (int nh = 0; nh < 2; ++nh)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int token = tn * TILE + nh * 128 + l.wc * 32 + j * 16 + l.fr;
      if constexpr (!DL) {
        float m = -INFINITY, s = 0.f;
#pragma unroll
        for (int mh = 0; mh < 2; ++mh)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float z = acc[mh][nh][i][j][e] * sc;
              if (!whole && vb + mh * 128 + i * 16 + e >= vn) z = -INFINITY;
              acc[mh][nh][i][j][e] = z;
              m = fmaxf(m, z);
            }
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int mh = 0; mh < 2; ++mh)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f(acc[mh][nh][i][j][e] - base);
        merge(m, s, __shfl_xor(m, 16, 64), __shfl_xor(s, 16, 64));
        merge(m, s, __shfl_xor(m, 32, 64), __shfl_xor(s, 32, 64));
        if (l.fq == 0 && token < rows) part[(size_t)(2 * tv + l.wr) * n + token] = float2{m, s};
      } else {
        if (token >= rows) continue;
        const float f = factor[token], ls = lse[token];
        T* out = static_cast<T*>(dl) + (size_t)token * lddl + vb;
#pragma unroll
        for (int mh = 0; mh < 2; ++mh)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float g[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float q = __builtin_amdgcn_exp2f(acc[mh][nh][i][j][e] * sc - ls);
              g[e] = whole || vb + mh * 128 + i * 16 + e < vn ? f * q : 0.f;  // zeros pad the piece
            }
            *reinterpret_cast<u32x2*>(out + mh * 128 + i * 16) = u32x2{pack2<T>(g[0], g[1]), pack2<T>(g[2], g[3])};
          }
      }
    }
}

// dX^T tile: A = W (K = vocabulary, down the rows), B = dl (K along the rows).  The piece's
// vocabulary is split over blockIdx.y; each split owns its own fp32 sums, added to from piece
// to piece, so the order of every sum is fixed.
template <bool F16>
__global__ __launch_bounds__(THREADS) void k_dx(const void* __restrict__ w, long long ldw, const void* __restrict__ dl,
                                                long long lddl, int v0, int vn, int d, int dp,
                                                const int* __restrict__ count, int n, int per_split, int first,
                                                float* __restrict__ out) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int rows = count[0];
  const int tiles_d = (d + TILE - 1) / TILE, tiles_n = (rows + TILE - 1) / TILE, nwg = tiles_d * tiles_n;
  if ((int)blockIdx.x >= nwg) return;
  int td, tn;
  tile_of(blockIdx.x, nwg, tiles_d, tiles_n, &td, &tn);
  const int tid = threadIdx.x, k0 = blockIdx.y * per_split, k = min(vn - k0, per_split);
  const Panel<false> pa(w, ldw, td * TILE, d, v0 + k0, max(k, 0), tid);
  const Panel<true> pb(dl, lddl, tn * TILE, rows, k0, (max(k, 0) + 7) & ~7, tid);  // dl is padded with zeros
  Acc acc;
  product<F16, false, true>(acc, smem, pa, pb, (k + KT - 1) / KT, tid);
  const Lane l(tid);
  out += (size_t)blockIdx.y * n * dp;
#pragma unroll
  for (int nh = 0; nh < 2; ++nh)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int token = tn * TILE + nh * 128 + l.wc * 32 + j * 16 + l.fr;
      if (token >= rows) continue;
#pragma unroll
      for (int mh = 0; mh < 2; ++mh)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = td * TILE + mh * 128 + l.wr * 64 + i * 16 + l.fq * 4;
          if (c >= dp) continue;
          f32x4* at = reinterpret_cast<f32x4*>(out + (size_t)token * dp + c);
          f32x4 r = acc[mh][nh][i][j];
          if (!first) r += *at;
          *at = r;
        }
    }
}

// dW^T tile: A = Xc (K = tokens, down the rows), B = dl (K = tokens, down the rows).
template <bool F16>
__global__ __launch_bounds__(THREADS) void k_dw(const void* __restrict__ xc, long long ldxc,
                                                const void* __restrict__ dl, long long lddl, int v0, int vn, int d,
                                                const int* __restrict__ count, const float* __restrict__ scale,
                                                void* __restrict__ dw, int lddw) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using T = typename Type<F16>::T;
  const int rows = count[0];
  const int tiles_d = (d + TILE - 1) / TILE, tiles_v = (vn + TILE - 1) / TILE;
  int td, tv;
  tile_of(blockIdx.x, tiles_d * tiles_v, tiles_d, tiles_v, &td, &tv);
  const int tid = threadIdx.x;
  const Panel<false> pa(xc, ldxc, td * TILE, (int)(ldxc / 2), 0, rows, tid);
  const Panel<false> pb(dl, lddl, tv * TILE, (int)(lddl / 2), 0, rows, tid);
  Acc acc;
  product<F16, false, false>(acc, smem, pa, pb, (rows + KT - 1) / KT, tid);
  const Lane l(tid);
  const float sc = scale[0];
  const bool wide = (lddw & 3) == 0 && (reinterpret_cast<uintptr_t>(dw) & 7) == 0;
#pragma unroll
  for (int nh = 0; nh < 2; ++nh)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = tv * TILE + nh * 128 + l.wc * 32 + j * 16 + l.fr;
      if (row >= vn) continue;
      T* out = static_cast<T*>(dw) + (size_t)(v0 + row) * lddw;
#pragma unroll
      for (int mh = 0; mh < 2; ++mh)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = td * TILE + mh * 128 + l.wr * 64 + i * 16 + l.fq * 4;
          const f32x4 r = rows ? acc[mh][nh][i][j] * sc : f32x4{0.f, 0.f, 0.f, 0.f};
          if (wide && c + 4 <= d) {
            *reinterpret_cast<u32x2*>(out + c) = u32x2{pack2<T>(r[0], r[1]), pack2<T>(r[2], r[3])};
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (c + e < d) out[c + e] = (T)r[e];
          }
        }
    }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// Distillation: the teacher's probabilities over the listed ids, one wave a row.  An id below
// 0 is no entry.  A row with no entry, or none above -inf, has no loss (flag 0).
__global__ __launch_bounds__(256) void k_teacher(const long long* __restrict__ ids, const float* __restrict__ logits,
                                                 int n, int k, float inv_t, float* __restrict__ p,
                                                 int* __restrict__ flag) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= n) return;
  ids += (size_t)row * k;
  logits += (size_t)row * k;
  p += (size_t)row * k;
  float m = -INFINITY;
  bool any = false;
  for (int i = lane; i < k; i += 64)
    if (ids[i] >= 0) {
      const float t = logits[i] * inv_t;
      any |= t != -INFINITY;  // NaN counts: it has to show in the loss
      m = fmaxf(m, t);
    }
  m = wave_max(m);
  any = __any(any);
  if (m == -INFINITY) m = 0.f;
  float s = 0.f;
  for (int i = lane; i < k; i += 64) s += ids[i] >= 0 ? exp2f((logits[i] * inv_t - m) * LOG2E) : 0.f;
  s = wave_sum(s);
  for (int i = lane; i < k; i += 64)
    p[i] = any && ids[i] >= 0 ? exp2f((logits[i] * inv_t - m) * LOG2E) / s : 0.f;
  if (lane == 0) flag[row] = any;
}

// Packs the rows that have a loss into xc [rows][dp] (zeros behind d).  A block takes 16 rows
// and counts the kept rows before them itself, which needs no second launch for a scan (8192
// tokens: 512 blocks read at most 64 KiB of targets each, out of L2).
template <typename T>
__global__ __launch_bounds__(256) void k_gather(const T* __restrict__ x, long long ldx, int n, int d, int dp,
                                                const long long* __restrict__ target, long long ignore,
                                                const int* __restrict__ flag, T* __restrict__ xc,
                                                int* __restrict__ rowmap, int* __restrict__ posof,
                                                int* __restrict__ count, float* __restrict__ loss) {
  __shared__ int total[4], kept[16];
  const int row0 = blockIdx.x * 16, tid = threadIdx.x;
  int c = 0;
  if (flag) {
    for (int r = tid; r < row0; r += 256) c += flag[r] != 0;
  } else {
    for (int r = tid; r < row0; r += 256) c += target[r] != ignore;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o, 64);
  if ((tid & 63) == 0) total[tid >> 6] = c;
  if (tid < 16) {
    const int r = row0 + tid;
    kept[tid] = r < n && (flag ? flag[r] != 0 : target[r] != ignore);
  }
  __syncthreads();
  int pos = total[0] + total[1] + total[2] + total[3];
  const bool wide = (d & 7) == 0 && (ldx & 7) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  for (int i = 0; i < 16 && row0 + i < n; ++i) {
    const int r = row0 + i;
    if (!kept[i]) {
      if (tid == 0) {
        posof[r] = -1;
        if (loss) loss[r] = 0.f;
      }
      continue;
    }
    T* out = xc + (size_t)pos * dp;
    const T* in = x + (long long)r * ldx;
    if (wide) {
      for (int e = tid * 8; e < dp; e += 256 * 8)
        *reinterpret_cast<u32x4*>(out + e) = e < d ? *reinterpret_cast<const u32x4*>(in + e) : u32x4{0, 0, 0, 0};
    } else {
      for (int e = tid; e < dp; e += 256) out[e] = e < d ? in[e] : (T)0.f;
    }
    if (tid == 0) {
      rowmap[pos] = r;
      posof[r] = pos;
    }
    ++pos;
  }
  if (tid == 0 && row0 + 16 >= n) count[0] = pos;
}

// A copy of w with rows of dp elements, zeros behind d: for a w whose rows are not 16-byte
// aligned, or whose width is no multiple of 8.
template <typename T>
__global__ __launch_bounds__(256) void k_pad(const T* __restrict__ w, long long ldw, long long rows, int d, int dp,
                                             T* __restrict__ out) {
  for (long long r = blockIdx.x; r < rows; r += gridDim.x)
    for (int e = threadIdx.x; e < dp; e += 256) out[r * dp + e] = e < d ? w[r * ldw + e] : (T)0.f;
}

// zk[pos][j] = x . w[id], one wave a target.  A cross entropy target outside the vocabulary
// gives NaN, as does a listed id past its end; an id below 0 in a list is no entry.
template <typename T>
__global__ __launch_bounds__(256) void k_dots(const T* __restrict__ xc, int dp, const T* __restrict__ w,
                                              long long ldw, int dk, const long long* __restrict__ ids, int k,
                                              long long v, int distill, const int* __restrict__ rowmap,
                                              const int* __restrict__ count, float* __restrict__ zk) {
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int pos = (int)(item / k), j = (int)(item - (long long)pos * k), lane = threadIdx.x & 63;
  if (pos >= count[0]) return;
  const long long id = ids[(size_t)rowmap[pos] * k + j];
  float s = 0.f;
  if (id >= 0 && id < v) {
    const T* a = xc + (size_t)pos * dp;
    const T* b = w + id * ldw;
    for (int e = lane * 8; e < dk; e += 512) {
      typedef __attribute__((ext_vector_type(8))) T t8;
      const t8 p = *reinterpret_cast<const t8*>(a + e), q = *reinterpret_cast<const t8*>(b + e);
#pragma unroll
      for (int i = 0; i < 8; ++i) s += (float)p[i] * (float)q[i];
    }
    s = wave_sum(s);
  } else if (!distill || id >= 0) {
    s = NAN;
  }
  if (lane == 0) zk[(size_t)pos * k + j] = s;
}

// Joins the tiles' (max, sum) of 8 rows, 32 threads a row, and forms the rows' losses.
// lse is kept in the exponent's base 2.
__global__ __launch_bounds__(256) void k_loss(const float2* __restrict__ part, int parts, int n,
                                              const float* __restrict__ zk, const float* __restrict__ p, int k,
                                              const int* __restrict__ rowmap, const int* __restrict__ count, float sc,
                                              float t2, float* __restrict__ lse, float* __restrict__ rowloss,
                                              float* __restrict__ loss) {
  __shared__ float sm[32][8], ss[32][8], sd[32][8];
  const int r = threadIdx.x & 7, slice = threadIdx.x >> 3, pos = blockIdx.x * 8 + r, rows = count[0];
  if ((int)blockIdx.x * 8 >= rows) return;
  float m = -INFINITY, s = 0.f, dot = 0.f;
  if (pos < rows) {
    for (int i = slice; i < parts; i += 32) {
      const float2 c = part[(size_t)i * n + pos];
      merge(m, s, c.x, c.y);
    }
    // sum_k p (ln p - ln 2 (z sc - lse)) = sum_k p (ln p - ln 2 z sc) + ln 2 lse
    if (p) {
      const size_t row = (size_t)rowmap[pos] * k;
      for (int i = slice; i < k; i += 32) {
        const float q = p[row + i], z = zk[(size_t)pos * k + i];
        if (q > 0.f) dot += q * (logf(q) - LN2 * sc * z);
        else if (q != q || z != z) dot = NAN;
      }
    } else if (slice == 0) {
      dot = -LN2 * sc * zk[pos];
    }
  }
  sm[slice][r] = m;
  ss[slice][r] = s;
  sd[slice][r] = dot;
  __syncthreads();
  if (threadIdx.x < 8 && pos < rows) {
    for (int i = 1; i < 32; ++i) {
      merge(m, s, sm[i][r], ss[i][r]);
      dot += sd[i][r];
    }
    const float l = m + log2f(s), out = t2 * (dot + LN2 * l);
    lse[pos] = l;
    rowloss[pos] = out;
    if (loss) loss[rowmap[pos]] = out;
  }
}

// The sum or mean of the rows' losses in a fixed order; a batch without any loss has 0.
__global__ __launch_bounds__(1024) void k_reduce(const float* __restrict__ rowloss, const int* __restrict__ count,
                                                 int mean, float* __restrict__ loss) {
  __shared__ double sum[16];
  const int rows = count[0];
  double s = 0.;
  for (int i = threadIdx.x; i < rows; i += 1024) s += rowloss[i];
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) s += sum[i];
    loss[0] = (float)(mean ? s / max(rows, 1) : s);
  }
}

// factor[pos] = span * g / max|g|, scale = max|g| T / span: dl holds factor * (q - p), and the
// products are scaled once, in 32 bits.  span is 1 for bf16, which has an fp32 exponent, and
// 2^15 for fp16: |q - p| <= 1 stays below its largest value 65504, and a probability keeps
// its 11 bits down to 2^-29 instead of 2^-14.  A row whose loss is NaN gets NaN gradients.
__global__ __launch_bounds__(1024) void k_factor(const float* __restrict__ grad, long long ldg, int reduction,
                                                 const int* __restrict__ rowmap, const int* __restrict__ count,
                                                 const float* __restrict__ rowloss, float t, float span,
                                                 float* __restrict__ factor, float* __restrict__ scale) {
  __shared__ float top[16];
  const int rows = count[0];
  float m = 0.f;
  if (reduction == 0) {
    for (int i = threadIdx.x; i < rows; i += 1024) m = fmaxf(m, fabsf(grad[rowmap[i] * ldg]));
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int i = 0; i < 16; ++i) m = fmaxf(m, top[i]);
  } else {
    m = fabsf(grad[0]);
  }
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float g = grad[reduction == 0 ? rowmap[i] * ldg : 0];
    const float l = rowloss[i];
    factor[i] = l != l ? NAN : g == 0.f ? 0.f : g / m * span;
  }
  if (threadIdx.x == 0) scale[0] = m * t / span / (reduction == 2 ? (float)max(rows, 1) : 1.f);
}

// Puts the targets into the piece's dl: f (q - sum of the p of that id).  One wave a row.
template <typename T>
__global__ __launch_bounds__(256) void k_fix(const long long* __restrict__ ids, const float* __restrict__ p, int k,
                                             const float* __restrict__ zk, const float* __restrict__ lse,
                                             const float* __restrict__ factor, const int* __restrict__ rowmap,
                                             const int* __restrict__ count, float sc, long long v0, long long vn,
                                             T* __restrict__ dl, long long lddl) {
  const int pos = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (pos >= count[0]) return;
  const size_t row = (size_t)rowmap[pos] * k;
  for (int i = lane; i < k; i += 64) {
    const long long id = ids[row + i];
    if (id < v0 || id >= v0 + vn) continue;
    float sum = 1.f;
    bool firstone = true;
    if (p) {
      sum = 0.f;
      for (int o = 0; o < k; ++o)
        if (ids[row + o] == id) {
          sum += p[row + o];
          firstone &= o >= i;
        }
    }
    if (firstone)
      dl[(size_t)pos * lddl + (id - v0)] =
          (T)(factor[pos] * (__builtin_amdgcn_exp2f(zk[(size_t)pos * k + i] * sc - lse[pos]) - sum));
  }
}

// Joins the splits of dX, scales, rounds once, and puts zeros into the rows without a loss.
template <typename T>
__global__ __launch_bounds__(256) void k_dx_out(const float* __restrict__ part, int splits, int n, int d, int dp,
                                                const int* __restrict__ posof, const float* __restrict__ scale,
                                                T* __restrict__ dx) {
  const int per_row = (d + 1023) / 1024, row = blockIdx.x / per_row, pos = posof[row];
  const int c = ((blockIdx.x - row * per_row) * 256 + threadIdx.x) * 4;
  if (c >= d) return;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (pos >= 0) {
    for (int i = 0; i < splits; ++i)
      s += *reinterpret_cast<const f32x4*>(part + ((size_t)i * n + pos) * dp + c);
    s *= scale[0];
  }
  T* out = dx + (size_t)row * d + c;
  if ((d & 3) == 0) {
    *reinterpret_cast<u32x2*>(out) = u32x2{pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3])};
  } else {
    for (int e = 0; e < 4 && c + e < d; ++e) out[e] = (T)s[e];
  }
}

// Where the kernels read w: w itself, or its padded copy.
struct Weight {
  const void* at;
  long long ldb;  // row stride in bytes
  int dk;         // the width that is read
};

Weight weight_of(const tkl_args& a, int dp) {
  if (a.wc) return {a.wc, (long long)dp * 2, dp};
  return {a.w, a.ldw * 2, (int)a.d};
}

int padded(long long d) { return (int)((d + 63) / 64 * 64); }

int check(const tkl_args& a) {
  const char* bad = nullptr;
  if (a.n < 1 || a.n > (1 << 20)) bad = "tokens must be 1 to 2^20";
  else if (a.d < 1 || a.d > (1 << 16)) bad = "the width must be 1 to 65536";
  else if (a.v < 1 || a.v > (1 << 24)) bad = "the vocabulary must have 1 to 2^24 entries";
  else if (a.k < 1 || a.k > 1024) bad = "1 to 1024 targets a token";
  else if (!a.wc && ((a.d & 7) || (a.ldw & 7) || (reinterpret_cast<uintptr_t>(a.w) & 15)))
    bad = "w's rows are not 16-byte aligned and there is no room for a copy";
  else if (!a.wc && (a.ldw < a.d || a.ldw > (1 << 21))) bad = "w's row stride must be its width to 2^21 elements";
  else if (a.reduction < 0 || a.reduction > 2) bad = "reduction must be 0 to 2";
  else if (!(a.temperature > 0.f)) bad = "the temperature must be above 0";
  if (bad) {
    snprintf(g_err, sizeof(g_err), "%s", bad);
    return -1;
  }
  return 0;
}

hipError_t set_lds_limit() {
  static std::once_flag once[64];
  static hipError_t result[64];
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
  std::call_once(once[dev], [dev] {
    const void* fns[] = {
        reinterpret_cast<const void*>(&k_logits<false, false>), reinterpret_cast<const void*>(&k_logits<true, false>),
        reinterpret_cast<const void*>(&k_logits<false, true>),  reinterpret_cast<const void*>(&k_logits<true, true>),
        reinterpret_cast<const void*>(&k_dx<false>),            reinterpret_cast<const void*>(&k_dx<true>),
        reinterpret_cast<const void*>(&k_dw<false>),            reinterpret_cast<const void*>(&k_dw<true>)};
    for (const void* f : fns) {
      result[dev] = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
      if (result[dev] != hipSuccess) return;
    }
  });
  return result[dev];
}

unsigned blocks(long long items, long long per) { return (unsigned)((items + per - 1) / per); }

template <bool F16>
hipError_t forward(const tkl_args& a) {
  using T = typename Type<F16>::T;
  hipStream_t s = static_cast<hipStream_t>(a.stream);
  const int n = (int)a.n, d = (int)a.d, k = (int)a.k, dp = padded(a.d);
  const long long* ids = static_cast<const long long*>(a.ids);
  int *rowmap = static_cast<int*>(a.rowmap), *posof = static_cast<int*>(a.posof), *count = static_cast<int*>(a.count),
      *flag = a.distill ? static_cast<int*>(a.flag) : nullptr;
  float *p = a.distill ? static_cast<float*>(a.p) : nullptr, *each = a.reduction == 0 ? static_cast<float*>(a.loss) : nullptr;
  const float t = a.temperature, sc = LOG2E / t;
  if (a.distill) k_teacher<<<blocks(n, 4), 256, 0, s>>>(ids, static_cast<const float*>(a.teacher), n, k, 1.f / t, p, flag);
  k_gather<T><<<blocks(n, 16), 256, 0, s>>>(static_cast<const T*>(a.x), a.ldx, n, d, dp, ids, a.ignore, flag,
                                            static_cast<T*>(a.xc), rowmap, posof, count, each);
  if (a.wc)
    k_pad<T><<<(unsigned)std::min<long long>(a.v, 65536), 256, 0, s>>>(static_cast<const T*>(a.w), a.ldw, a.v, d, dp,
                                                                       static_cast<T*>(a.wc));
  const Weight w = weight_of(a, dp);
  const unsigned tiles_v = blocks(a.v, TILE), tiles_n = blocks(n, TILE);
  k_logits<F16, false><<<tiles_v * tiles_n, THREADS, LDS, s>>>(w.at, w.ldb, a.xc, (long long)dp * 2, 0, (int)a.v, w.dk,
                                                               count, n, sc, static_cast<float2*>(a.part), nullptr,
                                                               nullptr, nullptr, 0);
  k_dots<T><<<blocks((long long)n * k, 4), 256, 0, s>>>(static_cast<const T*>(a.xc), dp, static_cast<const T*>(w.at),
                                                        w.ldb / 2, w.dk, ids, k, a.v, a.distill, rowmap, count,
                                                        static_cast<float*>(a.zk));
  k_loss<<<blocks(n, 8), 256, 0, s>>>(static_cast<const float2*>(a.part), 2 * (int)tiles_v, n,
                                      static_cast<const float*>(a.zk), p, k, rowmap, count, sc, t * t,
                                      static_cast<float*>(a.lse), static_cast<float*>(a.rowloss), each);
  if (a.reduction)
    k_reduce<<<1, 1024, 0, s>>>(static_cast<const float*>(a.rowloss), count, a.reduction == 2,
                                static_cast<float*>(a.loss));
  return hipGetLastError();
}

template <bool F16>
hipError_t backward(const tkl_args& a) {
  using T = typename Type<F16>::T;
  hipStream_t s = static_cast<hipStream_t>(a.stream);
  const int n = (int)a.n, d = (int)a.d, k = (int)a.k, dp = padded(a.d);
  const long long* ids = static_cast<const long long*>(a.ids);
  const int *rowmap = static_cast<const int*>(a.rowmap), *count = static_cast<const int*>(a.count);
  const float* p = a.distill ? static_cast<const float*>(a.p) : nullptr;
  const float *lse = static_cast<const float*>(a.lse), *zk = static_cast<const float*>(a.zk);
  const float t = a.temperature, sc = LOG2E / t, span = F16 ? 32768.f : 1.f;
  float *factor = static_cast<float*>(a.factor), *scale = factor + n;
  k_factor<<<1, 1024, 0, s>>>(static_cast<const float*>(a.grad), a.ldg, a.reduction, rowmap, count,
                              static_cast<const float*>(a.rowloss), t, span, factor, scale);
  if (a.wc)
    k_pad<T><<<(unsigned)std::min<long long>(a.v, 65536), 256, 0, s>>>(static_cast<const T*>(a.w), a.ldw, a.v, d, dp,
                                                                       static_cast<T*>(a.wc));
  const Weight w = weight_of(a, dp);
  const unsigned tiles_n = blocks(n, TILE), tiles_d = blocks(d, TILE);
  const long long ldl = a.piece * 2;  // bytes of a row of dl
  for (long long v0 = 0; v0 < a.v; v0 += a.piece) {
    const int vn = (int)std::min(a.piece, a.v - v0);
    k_logits<F16, true><<<blocks(vn, TILE) * tiles_n, THREADS, LDS, s>>>(
        w.at, w.ldb, a.xc, (long long)dp * 2, (int)v0, (int)v0 + vn, w.dk, count, n, sc, nullptr, lse, factor, a.dl,
        a.piece);
    k_fix<T><<<blocks(n, 4), 256, 0, s>>>(ids, p, k, zk, lse, factor, rowmap, count, sc, v0, vn, static_cast<T*>(a.dl),
                                          a.piece);
    if (a.want & 1) {
      const int per = (int)blocks(blocks(vn, KT), a.splits) * KT;
      k_dx<F16><<<dim3(tiles_d * tiles_n, (unsigned)a.splits), THREADS, LDS, s>>>(
          w.at, w.ldb, a.dl, ldl, (int)v0, vn, w.dk, dp, count, n, per, v0 == 0, static_cast<float*>(a.dxpart));
    }
    if (a.want & 2)
      k_dw<F16><<<tiles_d * blocks(vn, TILE), THREADS, LDS, s>>>(a.xc, (long long)dp * 2, a.dl, ldl, (int)v0, vn, d,
                                                                 count, scale, a.dw, d);
  }
  if (a.want & 1)
    k_dx_out<T><<<blocks(d, 1024) * (unsigned)n, 256, 0, s>>>(static_cast<const float*>(a.dxpart), (int)a.splits,
                                                                   n, d, dp, static_cast<const int*>(a.posof), scale,
                                                                   static_cast<T*>(a.dx));
  return hipGetLastError();
}

int on_device(const tkl_args* a, hipError_t (*run)(const tkl_args&)) {
  if (check(*a)) return -1;
  int prev = 0;
  hipError_t e = hipGetDevice(&prev);
  if (e != hipSuccess) return set_err("hipGetDevice", e);
  if (prev != a->dev && (e = hipSetDevice(a->dev)) != hipSuccess) return set_err("hipSetDevice", e);
  e = set_lds_limit();
  if (e == hipSuccess) e = run(*a);
  if (prev != a->dev) {
    const hipError_t back = hipSetDevice(prev);
    if (e == hipSuccess) e = back;
  }
  return e == hipSuccess ? 0 : set_err("launch", e);
}

}  // namespace

// The caller's struct has to be this one.
extern "C" int tkl_args_size() { return (int)sizeof(tkl_args); }

// Both are queued on a->stream and wait for nothing.  0, or -1 / a HIP error (tkl_last_error).
extern "C" int tkl_forward(const tkl_args* a) { return on_device(a, a->f16 ? forward<true> : forward<false>); }

extern "C" int tkl_backward(const tkl_args* a) {
  if (a->piece < TILE || a->piece % TILE || a->piece > (1 << 24) || a->splits < 1 || a->splits > 1024) {
    snprintf(g_err, sizeof(g_err), "piece %lld must be a multiple of %d, splits %lld 1 to 1024", a->piece, TILE,
             a->splits);
    return -1;
  }
  return on_device(a, a->f16 ? backward<true> : backward<false>);
}
