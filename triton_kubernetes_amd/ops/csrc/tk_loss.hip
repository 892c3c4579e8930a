// Losses of a language model's output head on MI355X (gfx950): the logits z = X W^T of N tokens
// over a vocabulary of V leave the kernel that multiplies only as sums, or, where the caller has
// them kept between the passes, in 16 bits.
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
// Forward: one matrix product whose epilogue reduces every tile of the vocabulary to a maximum
// and a sum per token and leaves a cross entropy's targets' logits (k_logits<LSE>), a dot product
// per entry of a teacher's lists (k_dots), and a join over the tiles (k_loss).
// Backward, in pieces of the vocabulary: the logits' 16-bit derivative dl, from the same product
// again (k_logits<DL>), or from codes that the forward pass kept (k_dl, struct Codes); a
// teacher's targets are put in by k_fix; then dX += dl W and dW = dl^T X.
//
// dl is rounded to 16 bits, which costs each product about as much as the rounding of its result.
// Most of a row's derivative is at its targets, though, and one number's rounding does not average
// out: it is common to the row's whole part of a gradient, up to 1.57 times what rounding the result
// once costs, all told.  So what the targets lose (`lost`: of a cross entropy each, of a teacher's list
// RESIDUALS a row) is given back, to dX in fp32 (k_dx_out), to dW as steps more of its product (k_dw;
// k_list finds each tile's).  Errors, as multiples of rounding the exact gradients once: a cross
// entropy 1.00 (1.18 without, 4096 tokens), 64 entries of a teacher 1.16 (1.41), at most 1.35 seen.
// It costs a step 1 % (4096 x 4096 x 32768), where many tokens meet a small vocabulary up to 12 %
// (8192 x 512 x 1000).  A caller who wants less error has dl in two parts (k_logits<TWO>): what its
// rounding took is rounded to 16 bits too and multiplied in its turn, which leaves 2^-16 of dl in
// bf16, 2^-22 in fp16 (errors 1.000; 4096 x 4096 x 32768 1.55 times as long).
//
// Measured at bf16, 8192 tokens x 4096 x 131072: k_logits 6.4 ms forward and 6.6 backward, 1.38 and
// 1.33 PF (matrix pipe busy 69 and 64 % of the time, at 1.9 GHz), k_dx 6.75 ms and k_dw 7.0, 1.30 and
// 1.26 PF; the rest 0.16 ms.  With the logits kept k_logits 6.5 ms and k_dl 0.72 ms, 5.9 TB/s, instead.
// The products are bound by the matrix pipe and LDS together, about 2050 cycles of each in a step
// of 64 that takes 2800 to 3100.
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

// One call's tensors and sizes (ops/loss.py packs the same fields in the same order).
struct tkl_args {
  long long n, d, v, k;        // tokens, width, vocabulary, targets per token
  long long ldx, ldw, ldg;     // row strides of x and w, stride of the upstream gradient (elements)
  long long ignore;            // cross entropy: the target that means "no loss"
  long long piece, fill;       // backward: vocabulary entries per piece, workgroups that fill the chip with dX
  int dev, f16, distill, reduction;  // reduction 0 none, 1 sum, 2 mean
  float temperature;
  int want;                    // backward: 1 dX, 2 dW, 3 both
  int small;                   // products in small tiles: 1 the logits, 2 dX, 4 dW; 8: dl in two parts
  int parts;                   // backward: of the tokens for dW; more than 1 only where there is one piece
  const void *x, *w, *ids, *teacher, *grad;
  void *loss, *kept;           // kept: from forward to backward (struct Kept)
  void *room;                  // forward: the tiles' maxima and sums; backward: dl, sums of dX, factors
  void *codes;                 // from forward to backward: the logits in 16 bits (struct Codes), or null
  void *wc;                    // a padded copy of w, where w's rows are not 16-byte aligned; forward makes it
  void *dx, *dw;
  void* stream;
};

namespace {

constexpr int KT = 64;  // K elements of a step (128 bytes of a row)
constexpr int MAX_TARGETS = 1024;
constexpr int RESIDUALS = 4;  // entries of a teacher's list whose rounding is made good; 1 of a cross entropy
constexpr float LARGE = 0.125f;  // |q - p| from which it is: at most 16 of a row
constexpr int FEW_ROWS = 512;  // up to which each tile of dW looks for its targets among all (a launch less)

// The two tilings of the matrix products.  A fragment is 16 x 16; a lane of a wave holds rows
// row(mf) + (lane / 16) * 4 + 0..3 and column col(nf) + lane % 16 of fragment (mf, nf).
struct Big {  // 8 waves, the schedule of product_big
  static constexpr int BM = 256, BN = 256, THREADS = 512, MF = 8, NF = 4, WAVES_M = 2,
                       LDS = 256 * (256 * 2 + 16) + 4096;  // the tile on its way out and sums; steps take 128 KiB
  static constexpr int SLOTS = 256;         // workgroups at a time
  static constexpr float SUM_COST = 4.3f;  // of a tile's sums: 116 ns, to 27 ns for a K step of 1
  static __device__ __forceinline__ int wave_m(int wid) { return wid >> 2; }
  static __device__ __forceinline__ int row(int mf, int wid) { return (mf >> 2) * 128 + (wid >> 2) * 64 + (mf & 3) * 16; }
  static __device__ __forceinline__ int col(int nf, int wid) { return (nf >> 1) * 128 + (wid & 3) * 32 + (nf & 1) * 16; }
};
struct Small {  // 4 waves, STEPS steps in LDS, two workgroups to a compute unit: for few tokens
  static constexpr int BM = 128, BN = 64, THREADS = 256, MF = 2, NF = 4, WAVES_M = 4, STEPS = 3,
                       LDS = STEPS * (BM + BN) * KT * 2;
  static constexpr int SLOTS = 512;
  static constexpr float SUM_COST = 1.f;
  static __device__ __forceinline__ int wave_m(int wid) { return wid; }
  static __device__ __forceinline__ int row(int mf, int wid) { return wid * 32 + mf * 16; }
  static __device__ __forceinline__ int col(int nf, int) { return nf * 16; }
};

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

// Block -> place in the order of the work, XCD-aware: workgroups go round-robin over the 8 XCDs,
// so XCD x takes the x-th run of the order, and what lies together in it shares panels in that
// XCD's L2.
__device__ __forceinline__ int run_of(int b, int nwg) {
  const int xcd = b & 7, q = nwg >> 3, rem = nwg & 7;
  return (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + (b >> 3);
}
// Place -> tile: 8 rows of tiles at a time, down the columns.
__device__ __forceinline__ void tile_of(int w, int tiles_m, int tiles_n, int* tm, int* tn) {
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

// 16 bytes a lane from two buffers (offset `voff`, zeros past their ends) to LDS at `lds` and
// `lds2` + 16 lane.
// In asm, because the compiler would wait for every copy in flight before each
// ds_read_b64_tr_b16 (2.25 instead of 1.83 ms for k_dx and k_dw at 8192 x 4096 x 32768); product() does the
// waiting.  A copy has no register output; it reads its operands when it is issued.
// (5 wait states before it: they would be needed had a vector instruction written the
// descriptor, which the compiler does not see to for asm; 1 between m0 and its use.)
__device__ __forceinline__ void copy16_twice(u32x4 one, u32x4 two, unsigned voff, unsigned lds, unsigned lds2) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
      "s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %4, 0 offen lds" ::"s"(lds),
      "s"(lds2), "v"(voff), "s"(one), "s"(two)
      : "memory", "m0");
}
__device__ __forceinline__ u32x4 buffer_of(const char* base, unsigned bytes) {
  const unsigned long long b = reinterpret_cast<unsigned long long>(base);
  // (the readfirstlanes are no instructions where the values are scalar already: they only
  // make the compiler keep the descriptor in scalar registers)
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)b), hi = __builtin_amdgcn_readfirstlane((unsigned)(b >> 32));
  return u32x4{lo, hi & 0xffffu, (unsigned)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}

// A panel of an operand, staged in images of ROWS rows by THREADS threads.  ALONG: a row of the
// panel lies along K (an image is ROWS rows of 128 bytes); else K is the matrix's row index (64
// rows of ROWS columns), and the fragments are transposed on their way out of LDS.
template <bool ALONG, int ROWS, int THREADS>
struct Panel;

// Rows along K: LDS image [ROWS][8 chunks of 16 bytes], chunk c of row r at c ^ (r/2 & 7) (the
// 16 rows of a fragment read land in 16 bank slots).
template <int ROWS, int THREADS>
struct Panel<true, ROWS, THREADS> {
  static constexpr int COPIES = ROWS * 8 / THREADS;
  const char* base;
  unsigned ld, kbytes;  // row stride, valid bytes of a row
  unsigned bytes;       // from base to the end of the last valid row (at most 256 rows: below 2^30)
  unsigned voff, chunk;

  __device__ __forceinline__ Panel(const void* m, long long ldb, int row0, int rows, int k0, int k, int tid) {
    base = static_cast<const char*>(m) + (long long)row0 * ldb + (long long)k0 * 2;
    ld = (unsigned)ldb;
    kbytes = k * 2;
    bytes = (min(rows - row0, 256) - 1) * ld + kbytes;
    const int r = tid >> 3;
    chunk = ((tid & 7) ^ ((r >> 1) & 7)) * 16;
    voff = r * ld + chunk;
  }
  // this thread's copies of step t, rows h * ROWS on, to LDS at dst (of this wave)
  __device__ __forceinline__ void stage(int t, int h, unsigned dst) const {
    const unsigned k = t * (KT * 2), v = k + chunk < kbytes ? voff : FAR;  // past the row's end: zeros
    auto buffer = [&](int i) {
      const unsigned at = (h * ROWS + i * (THREADS / 8)) * ld + k;
      return buffer_of(base + at, max((int)(bytes - at), 0));  // (rows past the last one: at most 2^31 behind it)
    };
#pragma unroll
    for (int i = 0; i < COPIES; i += 2)
      copy16_twice(buffer(i), buffer(i + 1), v, dst + i * THREADS * 16, dst + (i + 1) * THREADS * 16);
  }
  // the 16 rows at r0 of an image, K chunk kk of 32
  __device__ __forceinline__ static u32x4 frag(const char* img, int r0, int kk, int lane) {
    const int r = r0 + (lane & 15), c = kk * 4 + (lane >> 4);
    return *reinterpret_cast<const u32x4*>(img + r * 128 + ((c ^ ((r >> 1) & 7)) * 16));
  }
};

// K down the rows: LDS image [64 k][ROWS / 16 units of 32 bytes], unit u of row k at u ^ f(k).
// Half a wave reads rows 0-3 and 8-11 (mod 16) at once; f spreads them over the banks: with 256
// bytes a row all 8 differ, with 128 bytes those of equal parity do.  ds_read_b64_tr_b16 gives
// lane c of a 16-lane group the 4 values of column c from the 4 rows that the group reads.
template <int ROWS, int THREADS>
struct Panel<false, ROWS, THREADS> {
  static constexpr int COPIES = ROWS * 8 / THREADS, STRIDE = ROWS * 2, PER = ROWS / 8, KROWS = THREADS / PER;
  const char* base;
  int krows;
  unsigned ld, width;  // row stride, valid bytes of a row from base on
  unsigned voff;

  static __device__ __forceinline__ int f(int k) {
    return ROWS == 128 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2);
  }
  __device__ __forceinline__ Panel(const void* m, long long ldb, int col0, int cols, int k0, int k, int tid) {
    base = static_cast<const char*>(m) + (long long)k0 * ldb + (long long)col0 * 2;
    ld = (unsigned)ldb;
    krows = k;
    width = (cols - col0) * 2;
    const int r = tid / PER, c = tid % PER;
    voff = r * ld + ((((c >> 1) ^ f(r)) << 1) | (c & 1)) * 16;
  }
  __device__ __forceinline__ void stage(int t, int h, unsigned dst) const {
    auto buffer = [&](int i) {
      const int k = t * KT + i * KROWS, rows = min(krows - k, KROWS);
      const int end = rows > 0 ? (rows - 1) * (int)ld + (int)width - h * STRIDE : 0;  // at most 32 rows of 2^25 bytes
      return buffer_of(base + (unsigned long long)(unsigned)k * ld + h * STRIDE, max(end, 0));
    };
#pragma unroll
    for (int i = 0; i < COPIES; i += 2)
      copy16_twice(buffer(i), buffer(i + 1), voff, dst + i * THREADS * 16, dst + (i + 1) * THREADS * 16);
  }
  __device__ __forceinline__ static u32x4 frag(const char* img, int c0, int kk, int lane) {
    const int q = lane >> 4, l = lane & 15, k = kk * 32 + q * 8 + (l >> 2);
    const char* p = img + k * STRIDE + (((c0 >> 4) ^ f(q * 8 + (l >> 2))) * 32) + (l & 3) * 8;
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * STRIDE)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
};

__device__ __forceinline__ unsigned lds_of(const char* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}

template <class Tile, bool ALONG>
using PanelA = Panel<ALONG, 128, Tile::THREADS>;
template <class Tile, bool ALONG>
using PanelB = Panel<ALONG, Tile::BN == 256 ? 128 : Tile::BN, Tile::THREADS>;

// acc = one tile of A B^T over nk steps of 64.
template <class Tile>
using Acc = f32x4[Tile::MF][Tile::NF];

template <class Tile>
__device__ __forceinline__ void clear(Acc<Tile>& acc) {
#pragma unroll
  for (int i = 0; i < Tile::MF; ++i)
#pragma unroll
    for (int j = 0; j < Tile::NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// Three steps in LDS: while one is multiplied the next two are on their way.  (Six steps and one
// workgroup to a compute unit took as long at 1 x 4096 x 4096, 24 us.)
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
template <bool F16, bool AA, bool BA>
__device__ __forceinline__ void product_small(f32x4 (&acc)[2][4], char* smem, const Panel<AA, 128, 256>& pa,
                                              const Panel<BA, 64, 256>& pb, int nk, int tid) {
  using Tile = Small;
  if (nk <= 0) return;
  constexpr int BYTES = (Tile::BM + Tile::BN) * KT * 2, AB = Tile::BM * KT * 2, DEPTH = Tile::STEPS;
  constexpr int COPIES = Panel<AA, 128, 256>::COPIES + Panel<BA, 64, 256>::COPIES;
  const int lane = tid & 63, wid = tid >> 6;
  const unsigned lds0 = lds_of(smem) + __builtin_amdgcn_readfirstlane(wid) * 64 * 16;
  auto stage = [&](int t) {
    const unsigned dst = lds0 + t % DEPTH * BYTES;
    pa.stage(t, 0, dst);
    pb.stage(t, 0, dst + AB);
  };
  auto step = [&](int t) {
    const char *ia = smem + t % DEPTH * BYTES, *ib = ia + AB;
    u32x4 a[2][2], b[4][2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
      for (int i = 0; i < 2; ++i) a[i][kk] = Panel<AA, 128, 256>::frag(ia, Tile::row(i, wid), kk, lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j][kk] = Panel<BA, 64, 256>::frag(ib, Tile::col(j, wid), kk, lane);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = Type<F16>::mfma(a[i][kk], b[j][kk], acc[i][j]);
  };
#pragma unroll
  for (int t = 0; t < DEPTH - 1; ++t)
    if (t < nk) stage(t);
  for (int t = 0; t < nk; ++t) {
    // step t is there: younger are the DEPTH - 2 behind it, if they exist
    if (t + DEPTH - 1 <= nk) wait_copies<COPIES * (DEPTH - 2)>();
    else wait_copies<0>();
    barrier();  // for every wave, and the step before it has been read
    if (t + DEPTH - 1 < nk) stage(t + DEPTH - 1);
    step(t);
  }
}

// The schedule is the one of tk_gemm_screen.hip's k_gemm8: LDS holds half-tiles of two steps,
// a step is two phases of 32 matrix instructions per wave, and the wave groups wr = 0 and 1
// run one barrier apart, so that on every SIMD one wave feeds the matrix pipe while the other
// reads LDS and issues copies.  A wave reads twice as much of A as of B, so a panel down the rows,
// whose reads take twice as long, is better B; FLIP gives the tile transposed for that, with the
// lanes' 4 numbers along B.
template <bool F16, bool AA, bool BA, bool FLIP>
__device__ __forceinline__ void product_big(Acc<Big>& acc, char* smem, const PanelA<Big, AA>& pa,
                                        const PanelB<Big, BA>& pb, int nk, int tid) {
  constexpr int HBYTES = 128 * KT * 2;
  const int lane = tid & 63, wid = tid >> 6, wr = wid >> 2, wc = wid & 3;
  if (nk <= 0) return;

  const unsigned lds0 = lds_of(smem) + __builtin_amdgcn_readfirstlane(wid) * 64 * 16;
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
      for (int kk = 0; kk < 2; ++kk) a[i][kk] = PanelA<Big, AA>::frag(slot(t, mh), wr * 64 + i * 16, kk, lane);
  };
  auto read_b = [&](int t, int nh) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) b[nh][j][kk] = PanelB<Big, BA>::frag(slot(t, 2 + nh), wc * 32 + j * 16, kk, lane);
  };
  auto quad = [&](int mh, int nh) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
          acc[mh * 4 + i][nh * 2 + j] = FLIP ? Type<F16>::mfma(b[nh][j][kk], a[i][kk], acc[mh * 4 + i][nh * 2 + j])
                                             : Type<F16>::mfma(a[i][kk], b[nh][j][kk], acc[mh * 4 + i][nh * 2 + j]);
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
        for (int j = 0; j < 2; ++j) asm volatile("" : "+v"(acc[mh * 4 + i][nh * 2 + j]));
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

// (MORE: added to what acc holds, after a barrier, for LDS still holds the product before)
template <class Tile, bool F16, bool AA, bool BA, bool FLIP = false, bool MORE = false>
__device__ __forceinline__ void multiply(Acc<Tile>& acc, char* smem, const PanelA<Tile, AA>& pa,
                                         const PanelB<Tile, BA>& pb, int nk, int tid) {
  if constexpr (MORE) __syncthreads();
  else clear<Tile>(acc);
  if constexpr (Tile::BM == 256) product_big<F16, AA, BA, FLIP>(acc, smem, pa, pb, nk, tid);
  else product_small<F16, AA, BA>(acc, smem, pa, pb, nk, tid);
}

// (m, s) of a softmax: maximum and sum of exp2(. - m).  An empty side has m = -inf, s = 0.
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float a = m == top ? 1.f : exp2f(m - top), b = m2 == top ? 1.f : exp2f(m2 - top);
  s = s * a + s2 * b;
  m = top;
}

// A tile on its way out: column c of it is a row of the matrix, BM numbers of 16 bits, which go
// through LDS so that 16 (or 32) lanes store a whole row 16 bytes each.  (Straight out of the
// fragments, 4 lanes to 32 bytes of a row: 427 us for 388 of the logits' derivative at
// 1217 x 288 x 242340, 58 for 26 of w's gradient at 30 x 927 x 19663, whose rows start anywhere.)
template <class Tile, typename T>
struct Outgoing {
  static constexpr int STRIDE = Tile::BM * 2 + 16, PER = Tile::BM / 8;
  static constexpr int BYTES = Tile::BN * STRIDE;
  static_assert(BYTES + Tile::WAVES_M * Tile::BN * 8 <= Tile::LDS, "the tile and its sums fit");
  static __device__ __forceinline__ void put(char* smem, int col, int row, unsigned ab, unsigned cd) {
    *reinterpret_cast<u32x2*>(smem + col * STRIDE + row * 2) = u32x2{ab, cd};
  }
  static __device__ __forceinline__ void put(char* smem, int col, int row, float a, float b, float c, float d) {
    put(smem, col, row, pack2<T>(a, b), pack2<T>(c, d));
  }
  // rows first .. first + count of `out`, from column c0 on, `width` of them
  static __device__ __forceinline__ void store(const char* smem, T* out, long long ld, long long first, int count, int c0,
                                               int width, int tid) {
    for (int i = tid; i < count * PER; i += Tile::THREADS) {
      const int r = i / PER, c = i % PER * 8;
      const u32x4 v = *reinterpret_cast<const u32x4*>(smem + r * STRIDE + c * 2);
      T* to = out + (first + r) * ld + c0 + c;
      if (c + 8 <= width) __builtin_memcpy(to, &v, 16);  // at any alignment
      else if (c < width) {
        typedef __attribute__((ext_vector_type(8))) T t8;
        const t8 e = __builtin_bit_cast(t8, v);
#pragma unroll
        for (int o = 0; o < 8; ++o)
          if (c + o < width) to[o] = e[o];
      }
    }
  }
};

// What the derivative dl = factor (q - p) of a packed row's logits is multiplied with, and the
// scale that the products are multiplied with afterwards, in 32 bits.  For the sum and the mean
// factor is the upstream gradient's sign times `span`; without a reduction it is the row's
// upstream gradient itself, or for fp16 span * that / the largest one's magnitude, from k_factor.
// span is 1 for bf16, which has fp32's exponents, and 2^15 for fp16: |q - p| <= 1 stays below
// its largest value 65504, and a probability keeps its 11 bits down to 2^-29 instead of 2^-14.
// A row whose loss is NaN gets NaN gradients.
template <bool F16>
struct Upstream {
  const float *grad, *rowloss, *factor;  // factor[n] is the scale that goes with them
  const int *rowmap, *count;
  long long ldg;
  int reduction, n;
  float t;
  static constexpr float SPAN = F16 ? 32768.f : 1.f;

  __device__ __forceinline__ float of(int pos) const {
    const float l = rowloss[pos];
    if (l != l) return NAN;
    if (reduction == 0) return F16 ? factor[pos] : grad[rowmap[pos] * ldg];
    const float g = grad[0];
    return g > 0.f ? SPAN : g < 0.f ? -SPAN : g;
  }
  __device__ __forceinline__ float scale() const {
    if (reduction == 0) return F16 ? factor[n] : t;
    return fabsf(grad[0]) * t / SPAN / (reduction == 2 ? (float)max(count[0], 1) : 1.f);
  }
};

// A logit z (times log2(e) / T) in 16 bits, as its distance from the maximum M of its row within
// its tile: steps of 2^-12 down to M - 8, of 2^-10 to M - 24, of 2^-7 to M - 152, below which
// exp2 is 0 in fp32.  What a step's half is of q = exp2(z - lse), 8.5e-5, 3.4e-4 and 2.7e-3 of its
// value, joins the rounding of dl to bf16, 3.9e-3, or to fp16, 4.9e-4, whose numbers run out at
// 2^-29 of the largest (struct Upstream).
struct Codes {
  static constexpr float UNIT = 4096.f / 65535.f;  // a distance of 1, of the largest code
  static __device__ __forceinline__ unsigned pack(float a, float b) {  // distances, in UNITs
    auto code = [](float d) {  // the least of the three lines
      return fminf(fminf(d, __builtin_fmaf(d, 1.f / 4, 24576.f / 65535.f)), __builtin_fmaf(d, 1.f / 32, 46080.f / 65535.f));
    };
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pknorm_u16(code(a), code(b)));
  }
  static __device__ __forceinline__ float distance(unsigned code) {
    constexpr float S = 1.f / 4096.f;
    const float c = (float)code;
    return fmaxf(fmaxf(c * S, __builtin_fmaf(c, 4 * S, -98304.f * S)), __builtin_fmaf(c, 32 * S, -1474560.f * S));
  }
  // [n][stride] codes, then [tiles][n] maxima and sums
  static __host__ __device__ long long stride(long long v) { return (v + 255) / 256 * 256; }
};

// z^T of Tile::BM vocabulary entries (A = W) by Tile::BN tokens (B = Xc), so that a lane holds
// many entries of few tokens and the softmax's sums need two shuffles a token.
// LSE: writes part[tile][token] = (max, sum); KEEP: and the logits' codes to `out`.  DL: writes
// f (q - p) in 16 bits to `out`, with a cross entropy's p; `targets` is null for a teacher's
// lists.  TWO: the same, and what that rounding took, in 16 bits, to `low`.  sc = log2(e) / T.
// `of_target` gets of a cross entropy's targets the logits (LSE, KEEP), out of the accumulators that
// the sums are made from, or what their derivative's rounding took (DL, TWO).
enum Mode { LSE, KEEP, DL, TWO };
template <class Tile, bool F16, Mode MODE>
__global__ __launch_bounds__(Tile::THREADS) void k_logits(const void* __restrict__ w, long long ldw,
                                                          const void* __restrict__ xc, long long ldxc, int v0,
                                                          int vend, int d, const int* __restrict__ count, int n,
                                                          float sc, float2* __restrict__ part,
                                                          const float* __restrict__ lse, Upstream<F16> up,
                                                          const int* __restrict__ targets, void* __restrict__ out,
                                                          long long ldout, float* __restrict__ of_target,
                                                          void* __restrict__ low) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using T = typename Type<F16>::T;
  const int rows = count[0];
  const int tiles_v = (vend - v0 + Tile::BM - 1) / Tile::BM, tiles_n = (rows + Tile::BN - 1) / Tile::BN;
  const int nwg = tiles_v * tiles_n;
  if ((int)blockIdx.x >= nwg) return;
  int tv, tn;
  tile_of(run_of(blockIdx.x, nwg), tiles_v, tiles_n, &tv, &tn);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, fr = lane & 15, fq = lane >> 4;
  const PanelA<Tile, true> pa(w, ldw, v0 + tv * Tile::BM, vend, 0, d, tid);
  const PanelB<Tile, true> pb(xc, ldxc, tn * Tile::BN, rows, 0, d, tid);
  Acc<Tile> acc;
  multiply<Tile, F16, true, true>(acc, smem, pa, pb, (d + KT - 1) / KT, tid);

  const int vb = tv * Tile::BM + fq * 4;  // the lane's entries are vb + row(i) + 0..3, in the piece
  const int vn = vend - v0;
  const bool whole = (tv + 1) * Tile::BM <= vn;
  const int first = tn * Tile::BN, here = min(Tile::BN, rows - first);
  if constexpr (MODE == LSE || MODE == KEEP) {
    if (targets) {
#pragma unroll
      for (int j = 0; j < Tile::NF; ++j) {
        const int token = first + Tile::col(j, wid) + fr, target = token < rows ? targets[token] - v0 - vb : -Tile::BM;
        if ((unsigned)(target + 12) < Tile::BM + 12u) {  // (vb is up to 12 past the tile's start)
#pragma unroll
          for (int i = 0; i < Tile::MF; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (Tile::row(i, wid) + e == target) of_target[token] = acc[i][j][e];
        }
      }
    }
    barrier();  // LDS has been read
    float2* sums = reinterpret_cast<float2*>(smem + Outgoing<Tile, T>::BYTES);  // [WAVES_M][BN]
#pragma unroll
    for (int j = 0; j < Tile::NF; ++j) {
      float m = -INFINITY, s = 0.f;
      if (!whole) {
#pragma unroll
        for (int i = 0; i < Tile::MF; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (vb + Tile::row(i, wid) + e >= vn) acc[i][j][e] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < Tile::MF; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) m = fmaxf(m, acc[i][j][e]);
      m *= sc;
      const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < Tile::MF; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], sc, -base));
      merge(m, s, __shfl_xor(m, 16, 64), __shfl_xor(s, 16, 64));
      merge(m, s, __shfl_xor(m, 32, 64), __shfl_xor(s, 32, 64));
      if (fq == 0) sums[Tile::wave_m(wid) * Tile::BN + Tile::col(j, wid) + fr] = float2{m, s};
    }
    __syncthreads();
    if (tid < here) {
      float2 c = sums[tid];
#pragma unroll
      for (int o = 1; o < Tile::WAVES_M; ++o) merge(c.x, c.y, sums[o * Tile::BN + tid].x, sums[o * Tile::BN + tid].y);
      part[(size_t)tv * n + first + tid] = c;
    }
    if constexpr (MODE == KEEP) {
#pragma unroll
      for (int j = 0; j < Tile::NF; ++j) {
        const int col = Tile::col(j, wid) + fr;
        float m = sums[col].x;
#pragma unroll
        for (int o = 1; o < Tile::WAVES_M; ++o) m = fmaxf(m, sums[o * Tile::BN + col].x);
        m *= Codes::UNIT;
#pragma unroll
        for (int i = 0; i < Tile::MF; ++i) {
          float d[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) d[e] = __builtin_fmaf(acc[i][j][e], -sc * Codes::UNIT, m);
          Outgoing<Tile, T>::put(smem, col, Tile::row(i, wid) + fq * 4, Codes::pack(d[0], d[1]), Codes::pack(d[2], d[3]));
        }
      }
      __syncthreads();
      Outgoing<Tile, T>::store(smem, static_cast<T*>(out), ldout, first, here, tv * Tile::BM, Tile::BM, tid);
    }
  } else {
    __syncthreads();  // LDS has been read
#pragma unroll
    for (int j = 0; j < Tile::NF; ++j) {
      const int token = tn * Tile::BN + Tile::col(j, wid) + fr;
      const bool there = token < rows;
      const float f = there ? up.of(token) : 0.f, ls = there ? lse[token] : 0.f;
      const int target = there && targets ? targets[token] - v0 - vb : -1;
#pragma unroll
      for (int i = 0; i < Tile::MF; ++i) {
        const int at = Tile::row(i, wid);
        float g[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = f * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], sc, -ls));
        if ((unsigned)(target - at) < 4u) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (at + e == target) {
              g[e] -= f;
              of_target[token] = g[e] - (float)(T)g[e];
            }
        }
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (vb + at + e >= vn) g[e] = 0.f;  // zeros pad the piece
        }
        Outgoing<Tile, T>::put(smem, Tile::col(j, wid) + fr, at + fq * 4, g[0], g[1], g[2], g[3]);
        if constexpr (MODE == TWO) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = g[e] - (float)(T)g[e];
        }
      }
    }
    __syncthreads();
    Outgoing<Tile, T>::store(smem, static_cast<T*>(out), ldout, first, here, tv * Tile::BM, Tile::BM, tid);
    if constexpr (MODE == TWO) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < Tile::NF; ++j)
#pragma unroll
        for (int i = 0; i < Tile::MF; ++i)
          Outgoing<Tile, T>::put(smem, Tile::col(j, wid) + fr, Tile::row(i, wid) + fq * 4, acc[i][j][0], acc[i][j][1],
                                 acc[i][j][2], acc[i][j][3]);
      __syncthreads();
      Outgoing<Tile, T>::store(smem, static_cast<T*>(low), ldout, first, here, tv * Tile::BM, Tile::BM, tid);
    }
  }
}

// The kept logits' codes of a piece -> f (q - p) in 16 bits, as k_logits<DL> writes it.  A block
// takes 2048 entries of a row, 8 a thread; `at` and `zt` are the target and its logit of a cross
// entropy's row, whose q - 1 has to be better than a code is.  zeros pad the piece.
template <class Tile, bool F16>
__global__ __launch_bounds__(256) void k_dl(const unsigned short* __restrict__ codes, long long ldc,
                                            const float2* __restrict__ part, int n, int v0, int vn, float sc,
                                            const float* __restrict__ lse, Upstream<F16> up, const int* __restrict__ at,
                                            const float* __restrict__ zt, void* __restrict__ dl, long long lddl,
                                            float* __restrict__ lost) {
  using T = typename Type<F16>::T;
  const int per_row = (int)((lddl + 2047) / 2048), pos = blockIdx.x / per_row;
  const int c = ((blockIdx.x - pos * per_row) * 256 + threadIdx.x) * 8;
  if (pos >= up.count[0] || c >= lddl) return;
  u32x4 out = {0, 0, 0, 0};
  if (c < vn) {
    const u32x4 in = *reinterpret_cast<const u32x4*>(codes + pos * ldc + v0 + c);
    const float f = up.of(pos), ls = lse[pos], m = part[(size_t)((v0 + c) / Tile::BM) * n + pos].x - ls;
    const int target = (at ? at[pos] : -1) - v0 - c;
    float g[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = Codes::distance(in[e / 2] >> (e % 2 * 16) & 0xffffu);
      g[e] = c + e < vn ? f * __builtin_amdgcn_exp2f(m - d) : 0.f;
    }
    if ((unsigned)target < 8u) {
      const float t = f * (__builtin_amdgcn_exp2f(__builtin_fmaf(zt[pos], sc, -ls)) - 1.f);
      lost[pos] = t - (float)(T)t;
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = e == target ? t : g[e];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = pack2<T>(g[2 * i], g[2 * i + 1]);
  }
  *reinterpret_cast<u32x4*>(static_cast<T*>(dl) + pos * lddl + c) = out;
}

// Into how many parts the vocabulary is split for dX of `rows` packed rows, so that the last round
// of tiles over the compute units is as full as the others: of the most parts that 1, 2 or 3 rounds
// hold (`fill` workgroups at most, 512 entries of a piece or more each) those that cost least, a
// round's products and a tile's fp32 sums, written and read once more.  Only the device knows `rows`;
// k_dx leaves what it found to k_dx_out (`splits`), which has to read just as many sums.
template <class Tile>
__device__ __forceinline__ int splits_of(int rows, int d, int fill, int piece) {
  const int tiles = ((d + Tile::BM - 1) / Tile::BM) * ((rows + Tile::BN - 1) / Tile::BN);
  const int most = tiles ? min(fill / tiles, piece / 512) : 1;
  int best = 1;
  float least = INFINITY;
  for (int round = 1; round <= 3; ++round) {
    const int s = max(1, min(round * Tile::SLOTS / max(tiles, 1), most));
    const float cost = (float)((tiles * s + Tile::SLOTS - 1) / Tile::SLOTS) * piece / s + Tile::SUM_COST * tiles * s;
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

// dX^T tile of W (K = vocabulary, down the rows) and dl (K along the rows).  Each split owns
// its own fp32 sums [rows][dp], added to from piece to piece, so the order of every sum is fixed.
template <class Tile, bool F16>
__global__ __launch_bounds__(Tile::THREADS) void k_dx(const void* __restrict__ w, long long ldw,
                                                      const void* __restrict__ dl, long long lddl, int v0, int vn,
                                                      int d, int dp, const int* __restrict__ count, int fill,
                                                      int first, float* __restrict__ out, int* __restrict__ chosen) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int rows = count[0], splits = splits_of<Tile>(rows, d, fill, (int)(lddl / 2));
  const int tiles_d = (d + Tile::BM - 1) / Tile::BM, tiles_n = (rows + Tile::BN - 1) / Tile::BN;
  const int tiles = tiles_d * tiles_n, nwg = tiles * splits;
  if (blockIdx.x == 0 && threadIdx.x == 0) *chosen = splits;
  if ((int)blockIdx.x >= nwg) return;
  const int place = run_of(blockIdx.x, nwg), split = place / tiles;
  int td, tn;
  tile_of(place - split * tiles, tiles_d, tiles_n, &td, &tn);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int per_split = ((vn + KT - 1) / KT + splits - 1) / splits * KT;
  const int k0 = split * per_split, k = max(0, min(vn - k0, per_split));
  constexpr bool BIG = Tile::BM == Tile::BN;  // W as B (8192 x 4096 x 32768: 1684 us, 1837 with it as A)
  Acc<Tile> acc;
  if constexpr (BIG) {
    const PanelA<Tile, true> pa(dl, lddl, tn * Tile::BM, rows, k0, (k + 7) & ~7, tid);  // dl is padded with zeros
    const PanelB<Tile, false> pb(w, ldw, td * Tile::BN, d, v0 + k0, k, tid);
    multiply<Tile, F16, true, false, true>(acc, smem, pa, pb, (k + KT - 1) / KT, tid);
  } else {
    const PanelA<Tile, false> pa(w, ldw, td * Tile::BM, d, v0 + k0, k, tid);
    const PanelB<Tile, true> pb(dl, lddl, tn * Tile::BN, rows, k0, (k + 7) & ~7, tid);
    multiply<Tile, F16, false, true>(acc, smem, pa, pb, (k + KT - 1) / KT, tid);
  }
  out += (size_t)split * rows * dp;
#pragma unroll
  for (int j = 0; j < Tile::NF; ++j) {
#pragma unroll
    for (int i = 0; i < Tile::MF; ++i) {
      const int of_a = Tile::row(i, wid), of_b = Tile::col(j, wid);
      const int token = tn * Tile::BN + (BIG ? of_a : of_b) + (lane & 15);
      const int c = td * Tile::BM + (BIG ? of_b : of_a) + (lane >> 4) * 4;
      if (token >= rows || c >= dp) continue;
      f32x4* at = reinterpret_cast<f32x4*>(out + (size_t)token * dp + c);
      f32x4 r = acc[i][j];
      if (!first) r += *at;
      *at = r;
    }
  }
}

// Xc^T [dp][np] of the packed rows, zeros behind them up to the next 64, in tiles of 64 x 64.
template <typename T>
__global__ __launch_bounds__(256) void k_transpose(const T* __restrict__ xc, int dp, const int* __restrict__ count,
                                                   T* __restrict__ xt, int np) {
  __shared__ __attribute__((aligned(16))) T tile[64][72];
  typedef __attribute__((ext_vector_type(8))) T t8;
  const int rows = count[0], c0 = blockIdx.x * 64, r0 = blockIdx.y * 64, at = threadIdx.x >> 3, unit = (threadIdx.x & 7) * 8;
  if (r0 >= rows) return;
#pragma unroll
  for (int h = 0; h < 64; h += 32) {
    u32x4 v = {0, 0, 0, 0};
    if (r0 + at + h < rows) v = *reinterpret_cast<const u32x4*>(xc + (size_t)(r0 + at + h) * dp + c0 + unit);
    *reinterpret_cast<u32x4*>(&tile[at + h][unit]) = v;
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 64; h += 32) {
    t8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = tile[unit + i][at + h];
    *reinterpret_cast<t8*>(xt + (size_t)(c0 + at + h) * np + r0 + unit) = v;
  }
}

// The entries (of all packed rows' `at`) whose vocabulary entry is in the piece, by BUCKET entries of it:
// those of bucket b are listed[starts[b] .. starts[b + 1]), in order.  A block finds those of its
// bucket, and how many are in the buckets before it, by looking at all.
constexpr int BUCKET = 256;
__global__ __launch_bounds__(1024) void k_list(const int* __restrict__ at, int residuals, const int* __restrict__ count,
                                               int v0, int vn, int* __restrict__ listed, int* __restrict__ starts) {
  __shared__ int before[16], found[16];
  const int rows = count[0];
  if (rows <= FEW_ROWS) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, entries = rows * residuals;
  const int lo = v0 + blockIdx.x * BUCKET, hi = min(lo + BUCKET, v0 + vn);
  const int per = (entries + 1023) / 1024, i0 = min(entries, tid * per), i1 = min(entries, i0 + per);
  int below = 0, mine = 0;
#pragma unroll 8
  for (int i = i0; i < i1; ++i) {
    const int t = at[i];
    below += t >= v0 && t < lo;
    mine += t >= lo && t < hi;
  }
  int upto = mine;  // of this wave's lanes up to this one
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int other = __shfl_up(upto, o, 64);
    if (lane >= o) upto += other;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) below += __shfl_xor(below, o, 64);
  if (lane == 63) found[wave] = upto;
  if (lane == 0) before[wave] = below;
  __syncthreads();
  int start = 0, to = upto - mine, total = 0;
  for (int o = 0; o < 16; ++o) {
    start += before[o];
    if (o < wave) to += found[o];
    total += found[o];
  }
  if (tid == 0) {
    starts[blockIdx.x] = start;
    if (blockIdx.x == gridDim.x - 1) starts[blockIdx.x + 1] = start + total;
  }
  if (!mine) return;
  for (int i = i0; i < i1; ++i) {
    const int t = at[i];
    if (t >= lo && t < hi) listed[start + to++] = i;
  }
}

// dW^T tile: A = Xc^T (K = tokens along the rows), B = dl (K = tokens, down the rows).  (With A down
// the rows of Xc its fragments have to be transposed on their way out of LDS too, which takes twice
// the time of a plain read: 1950 us for 1724 at 8192 x 4096 x 32768.  Small tiles do that, and save a
// launch: 21 us both ways at 8192 x 512 x 1000.)  Where dW has few tiles the tokens are split over
// blockIdx.y, and each part writes its fp32 sums [v][dp], which k_dw_out adds in order (8192 x 512 x
// 1000, 128 tiles: 86 us whole, 26 in 4 parts).
template <class Tile, bool F16, bool TWICE>
__global__ __launch_bounds__(Tile::THREADS) void k_dw(const void* __restrict__ xt, long long ldxt,
                                                      const void* __restrict__ xc, int dp, const void* __restrict__ dl,
                                                      long long lddl, int v0, int vn, int d, const int* __restrict__ count, Upstream<F16> up,
                                                      const int* __restrict__ at, const float* __restrict__ lost,
                                                      int residuals, void* __restrict__ dw, int lddw,
                                                      float* __restrict__ sums, const void* __restrict__ low,
                                                      const int* __restrict__ listed, const int* __restrict__ starts) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using T = typename Type<F16>::T;
  const int rows = count[0], per = ((rows + KT - 1) / KT + gridDim.y - 1) / gridDim.y * KT;
  const int k0 = blockIdx.y * per, k = max(0, min(rows - k0, per));
  const int tiles_d = (d + Tile::BM - 1) / Tile::BM, tiles_v = (vn + Tile::BN - 1) / Tile::BN;
  int td, tv;
  tile_of(run_of(blockIdx.x, tiles_d * tiles_v), tiles_d, tiles_v, &td, &tv);
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const PanelB<Tile, false> pb(dl, lddl, tv * Tile::BN, (int)(lddl / 2), k0, k, tid);
  auto of_low = [&] { return PanelB<Tile, false>(low, lddl, tv * Tile::BN, (int)(lddl / 2), k0, k, tid); };
  Acc<Tile> acc;
  if constexpr (Tile::BM == Tile::BN) {
    const PanelA<Tile, true> pa(xt, ldxt, td * Tile::BM, dp, k0, (k + 7) & ~7, tid);
    multiply<Tile, F16, true, false>(acc, smem, pa, pb, (k + KT - 1) / KT, tid);
    if constexpr (TWICE)
      multiply<Tile, F16, true, false, false, true>(acc, smem, pa, of_low(), (k + KT - 1) / KT, tid);
  } else {
    const PanelA<Tile, false> pa(xc, 2 * dp, td * Tile::BM, dp, k0, k, tid);
    multiply<Tile, F16, false, false>(acc, smem, pa, pb, (k + KT - 1) / KT, tid);
    if constexpr (TWICE)
      multiply<Tile, F16, false, false, false, true>(acc, smem, pa, of_low(), (k + KT - 1) / KT, tid);
  }

  // What dl's rounding took from the targets among this tile's rows: a window of entries at a time, of all
  // of them where they are few, else of those that k_list found for these 256 rows.  The hits of a window
  // are put together in order; 64 of them are a step more of the product, of their rows of Xc with a
  // matrix that has each one's rest at its column.  (By vector instructions, a hit at a time, 8192 x 4096 x
  // 1536 with 1400 hits a tile took 770 us instead of 550 without any of this.)
  if constexpr (!TWICE) {
    constexpr int WAVES = Tile::THREADS / 64, PER = Tile::BM / 8;
    using Image = Panel<false, 128, Tile::THREADS>;  // of the hits' rows of Xc, 128 columns each
    int* hit_pos = reinterpret_cast<int*>(smem);  // [THREADS]
    int* hit_col = hit_pos + Tile::THREADS;
    float* hit_lost = reinterpret_cast<float*>(hit_col + Tile::THREADS);
    int* lengths = reinterpret_cast<int*>(hit_lost + Tile::THREADS);
    char* images = smem + 16384;
    static_assert(3 * Tile::THREADS * 4 + WAVES * 4 <= 16384, "the hits fit");
    static_assert(16384 + 64 * PER * 16 <= Tile::LDS, "the rows fit");
    const bool few = rows <= FEW_ROWS;
    const int bucket = tv * Tile::BN / BUCKET, start = few ? 0 : starts[bucket];
    const int entries = few ? rows * residuals : starts[bucket + 1] - start;
    const int share = (entries + (int)gridDim.y - 1) / (int)gridDim.y, end = min(entries, ((int)blockIdx.y + 1) * share);
    const int first = v0 + tv * Tile::BN, width = min(Tile::BN, vn - tv * Tile::BN);
    for (int i0 = blockIdx.y * share; i0 < end; i0 += Tile::THREADS) {
      const int i = i0 + tid, e = i >= end ? -1 : few ? i : listed[start + i], v = e < 0 ? -1 : at[e] - first;
      const bool here = v >= 0 && v < width;
      const unsigned long long mask = __ballot(here);
      __syncthreads();  // LDS has been read
      if (lane == 0) lengths[wid] = __popcll(mask);
      __syncthreads();
      int slot = __popcll(mask & ((1ull << lane) - 1)), total = 0;
      for (int o = 0; o < WAVES; ++o) {
        if (o < wid) slot += lengths[o];
        total += lengths[o];
      }
      if (here) {
        hit_pos[slot] = e / residuals;
        hit_col[slot] = v;
        hit_lost[slot] = lost[e];
      }
      if (tid >= total) hit_col[tid] = -1;  // none
      __syncthreads();
      for (int b = 0; b < total; b += 64) {
        if (b) __syncthreads();
        for (int x = tid; x < 64 * PER; x += Tile::THREADS) {
          const int k = x / PER, c = x % PER, unit = c & 15;
          u32x4 v8 = {0, 0, 0, 0};
          if (b + k < total && td * Tile::BM + c * 8 < dp)
            v8 = *reinterpret_cast<const u32x4*>(static_cast<const T*>(xc) + (size_t)hit_pos[b + k] * dp + td * Tile::BM + c * 8);
          *reinterpret_cast<u32x4*>(images + (c >> 4) * 64 * Image::STRIDE + k * Image::STRIDE +
                                    ((((unit >> 1) ^ Image::f(k)) << 1) | (unit & 1)) * 16) = v8;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          u32x4 x[Tile::MF];
#pragma unroll
          for (int m = 0; m < Tile::MF; ++m)
            x[m] = Image::frag(images + (Tile::row(m, wid) >> 7) * 64 * Image::STRIDE, Tile::row(m, wid) & 127, kk, lane);
          int cols[8];
          float rest[8];
#pragma unroll
          for (int o = 0; o < 8; ++o) {
            cols[o] = hit_col[b + kk * 32 + (lane >> 4) * 8 + o];
            rest[o] = hit_lost[b + kk * 32 + (lane >> 4) * 8 + o];
          }
#pragma unroll
          for (int j = 0; j < Tile::NF; ++j) {
            const int own = Tile::col(j, wid) + (lane & 15);
            bool any = false;
            u32x4 r;
#pragma unroll
            for (int o = 0; o < 4; ++o) {
              const bool p = cols[2 * o] == own, q = cols[2 * o + 1] == own;
              any |= p || q;
              r[o] = pack2<T>(p ? rest[2 * o] : 0.f, q ? rest[2 * o + 1] : 0.f);
            }
            if (!__any(any)) continue;
#pragma unroll
            for (int m = 0; m < Tile::MF; ++m) acc[m][j] = Type<F16>::mfma(x[m], r, acc[m][j]);
          }
        }
      }
    }
  }
  if (gridDim.y > 1) {
    sums += (size_t)blockIdx.y * vn * dp;
#pragma unroll
    for (int j = 0; j < Tile::NF; ++j) {
      const int v = tv * Tile::BN + Tile::col(j, wid) + (lane & 15);
#pragma unroll
      for (int i = 0; i < Tile::MF; ++i) {
        const int c = td * Tile::BM + Tile::row(i, wid) + (lane >> 4) * 4;
        if (v < vn && c < dp) *reinterpret_cast<f32x4*>(sums + (size_t)v * dp + c) = acc[i][j];
      }
    }
    return;
  }
  const float sc = up.scale();
  __syncthreads();  // LDS has been read
#pragma unroll
  for (int j = 0; j < Tile::NF; ++j)
#pragma unroll
    for (int i = 0; i < Tile::MF; ++i) {
      const f32x4 r = rows ? acc[i][j] * sc : f32x4{0.f, 0.f, 0.f, 0.f};
      Outgoing<Tile, T>::put(smem, Tile::col(j, wid) + (lane & 15), Tile::row(i, wid) + (lane >> 4) * 4, r[0], r[1], r[2],
                             r[3]);
    }
  __syncthreads();
  Outgoing<Tile, T>::store(smem, static_cast<T*>(dw), lddw, v0 + tv * Tile::BN, min(Tile::BN, vn - tv * Tile::BN),
                           td * Tile::BM, d - td * Tile::BM, tid);
}

// Joins the parts of dW: 4 columns of a row a thread.
template <bool F16>
__global__ __launch_bounds__(256) void k_dw_out(const float* __restrict__ sums, int parts, long long v, int d, int dp,
                                                Upstream<F16> up, void* __restrict__ dw) {
  using T = typename Type<F16>::T;
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x, row = item / (dp / 4);
  const int c = (int)(item - row * (dp / 4)) * 4;
  if (row >= v || c >= d) return;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (up.count[0]) {
#pragma unroll 4
    for (int i = 0; i < parts; ++i) s += *reinterpret_cast<const f32x4*>(sums + (i * v + row) * dp + c);
    s *= up.scale();
  }
  T* out = static_cast<T*>(dw) + row * d + c;
  for (int e = 0; e < 4 && c + e < d; ++e) out[e] = (T)s[e];
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
      any |= logits[i] != -INFINITY;  // NaN counts: it has to show in the loss
      m = fmaxf(m, logits[i]);
    }
  m = wave_max(m);
  any = __any(any);
  if (m == -INFINITY) m = 0.f;
  // (the difference before the division: a list of the type's lowest value is uniform at any T)
  const float sc = inv_t * LOG2E;
  float s = 0.f;
  for (int i = lane; i < k; i += 64) s += ids[i] >= 0 ? exp2f((logits[i] - m) * sc) : 0.f;
  s = wave_sum(s);
  for (int i = lane; i < k; i += 64) p[i] = any && ids[i] >= 0 ? exp2f((logits[i] - m) * sc) / s : 0.f;
  if (lane == 0) flag[row] = any;
}

// Packs the rows that have a loss into xc [rows][dp] (zeros behind d), and of a cross entropy the
// targets (`at`; one outside the vocabulary is -1, and its logit in `zk` NaN).  A wave takes `per` rows, and
// its block counts the kept rows before them itself, which needs no second launch for a scan
// (8192 tokens: 1024 blocks read at most 64 KiB of targets each, out of L2).
constexpr int MOST_PER = 32;
int gather_rows(int n) { return n <= 65536 ? 2 : (n + 32767) / 32768; }  // at most about 8192 blocks
template <typename T>
__global__ __launch_bounds__(256) void k_gather(const T* __restrict__ x, long long ldx, int n, int d, int dp,
                                                const long long* __restrict__ target, long long ignore,
                                                const int* __restrict__ flag, T* __restrict__ xc,
                                                int* __restrict__ rowmap, int* __restrict__ posof,
                                                int* __restrict__ count, float* __restrict__ loss, int per,
                                                long long v, int* __restrict__ at, float* __restrict__ zk) {
  __shared__ int total[4], kept[4 * MOST_PER];
  const int row0 = blockIdx.x * 4 * per, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int c = 0;
  if (flag) {
#pragma unroll 8
    for (int r = tid; r < row0; r += 256) c += flag[r] != 0;
  } else {
#pragma unroll 8
    for (int r = tid; r < row0; r += 256) c += target[r] != ignore;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o, 64);
  if (lane == 0) total[wave] = c;
  if (tid < 4 * per) {
    const int r = row0 + tid;
    kept[tid] = r < n && (flag ? flag[r] != 0 : target[r] != ignore);
  }
  __syncthreads();
  int pos = total[0] + total[1] + total[2] + total[3];
  if (tid == 0 && row0 + 4 * per >= n) {
    int all = pos;
    for (int i = 0; i < 4 * per; ++i) all += kept[i];
    count[0] = all;
    count[1] = 0;
  }
  for (int i = 0; i < wave * per; ++i) pos += kept[i];
  for (int i = wave * per; i < (wave + 1) * per; ++i) {
    const int r = row0 + i;
    if (r >= n) break;
    if (!kept[i]) {
      if (lane == 0) {
        posof[r] = -1;
        if (loss) loss[r] = 0.f;
      }
      continue;
    }
    T* out = xc + (size_t)pos * dp;
    const T* in = x + (long long)r * ldx;
#pragma unroll 8
    for (int e = lane * 8; e + 8 <= d; e += 512) {
      u32x4 v;
      __builtin_memcpy(&v, in + e, 16);  // at any alignment
      *reinterpret_cast<u32x4*>(out + e) = v;
    }
    for (int e = (d & ~7) + lane; e < dp; e += 64) out[e] = e < d ? in[e] : (T)0.f;
    if (lane == 0) {
      rowmap[pos] = r;
      posof[r] = pos;
      if (!flag) {
        const bool there = target[r] >= 0 && target[r] < v;
        at[pos] = there ? (int)target[r] : -1;
        if (!there) zk[pos] = NAN;
      }
    }
    ++pos;
  }
}

// A copy of w with rows of dp elements, zeros behind d: for a w whose rows are not 16-byte
// aligned, or whose width is no multiple of 8.  16 bytes a thread, read at any alignment.
template <typename T>
__global__ __launch_bounds__(256) void k_pad(const T* __restrict__ w, long long ldw, long long rows, int d, int dp,
                                             T* __restrict__ out) {
  const int per = dp / 8;
  const long long all = rows * per;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
    const long long r = i / per;
    const int e = (int)(i - r * per) * 8;
    u32x4 v = {0, 0, 0, 0};
    if (e + 8 <= d) {
      __builtin_memcpy(&v, w + r * ldw + e, 16);
    } else if (e < d) {
      typedef __attribute__((ext_vector_type(8))) T t8;
      t8 one;
#pragma unroll
      for (int o = 0; o < 8; ++o) one[o] = e + o < d ? w[r * ldw + e + o] : (T)0.f;
      v = __builtin_bit_cast(u32x4, one);
    }
    *reinterpret_cast<u32x4*>(out + r * dp + e) = v;
  }
}

// A teacher's lists: zk[pos][j] = x . w[id], one wave for 16 entries of a token.  By matrix instructions
// in the order of k_logits' steps, so that each is that kernel's logit to the bit: a loss is a
// difference of the two (a student that is sure of the same entry as its teacher had 4 times the
// plain form's error with sums of their own order).  An id below 0 is no entry.  (2048 tokens x 64
// entries of 2048: 81 to 87 us, 6.4 TB/s.)
template <bool F16>
__global__ __launch_bounds__(256) void k_dots(const void* __restrict__ xc, int dp, const void* __restrict__ w,
                                              long long ldw, int dk, const long long* __restrict__ ids, int k,
                                              long long v, const int* __restrict__ rowmap,
                                              const int* __restrict__ count, float* __restrict__ zk) {
  using T = typename Type<F16>::T;
  constexpr int SHARE = 16, AHEAD = 8;
  const int per_row = (k + SHARE - 1) / SHARE, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const long long items = (long long)count[0] * per_row;
  for (long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); i < items; i += (long long)gridDim.x * 4) {
    const int pos = (int)(i / per_row), j = (int)(i - (long long)pos * per_row) * SHARE;
    const long long* row = ids + (size_t)rowmap[pos] * k;
    const long long id = j + r < k ? row[j + r] : -1;
    const bool there = id >= 0 && id < v;
    const T* from = static_cast<const T*>(w) + (there ? id : 0) * ldw + q * 8;
    const T* x = static_cast<const T*>(xc) + (size_t)pos * dp + q * 8;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int e = 0; e < dk; e += 32 * AHEAD) {
      u32x4 a[AHEAD], b[AHEAD];
#pragma unroll
      for (int o = 0; o < AHEAD; ++o) {
        const bool in = e + o * 32 + q * 8 < dk;
        a[o] = in && there ? *reinterpret_cast<const u32x4*>(from + e + o * 32) : u32x4{0, 0, 0, 0};
        b[o] = in ? *reinterpret_cast<const u32x4*>(x + e + o * 32) : u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int o = 0; o < AHEAD; ++o) acc = Type<F16>::mfma(a[o], b[o], acc);
    }
    // every column has the 16 sums, 4 to a lane: column c of 4 writes its lanes' c-th
    const int own = j + q * 4 + r;
    if (r < 4 && own < k) {
      const float z = r == 0 ? acc[0] : r == 1 ? acc[1] : r == 2 ? acc[2] : acc[3];
      const long long of = row[own];
      zk[(size_t)pos * k + own] = of < 0 ? 0.f : of < v ? z : NAN;
    }
  }
}

// Joins the tiles' (max, sum) of 8 rows, 32 threads a row, and forms the rows' losses.  lse is kept in the
// exponent's base 2, but the losses take the targets' distance from the row's maximum m, exact but for
// one rounding, where a difference of lse and logit would have theirs:
//
//     log q = ln 2 ((z sc - m) - log2 sum_v exp2(z_v sc - m))
//
// With a reduction the block that ends last adds the rows' losses, always in the same order (`done` not
// null; the release that this takes of every block costs 60 us of 1024 blocks, so many rows have
// k_reduce).  A batch without any loss has 0.
__global__ __launch_bounds__(256) void k_loss(const float2* __restrict__ part, int parts, int n,
                                              const float* __restrict__ zk, const float* __restrict__ p, int k,
                                              const int* __restrict__ rowmap, const int* __restrict__ count, float sc,
                                              float t2, float* __restrict__ lse, float* __restrict__ rowloss,
                                              float* __restrict__ loss, int reduction, int* __restrict__ done) {
  __shared__ float sm[32][8], ss[32][8], sd[32][8];
  const int r = threadIdx.x & 7, slice = threadIdx.x >> 3, pos = blockIdx.x * 8 + r, rows = count[0];
  float m = -INFINITY, s = 0.f;
  if (pos < rows) {
#pragma unroll 4
    for (int i = slice; i < parts; i += 32) {
      const float2 c = part[(size_t)i * n + pos];
      merge(m, s, c.x, c.y);
    }
  }
  sm[slice][r] = m;
  ss[slice][r] = s;
  __syncthreads();
  m = sm[0][r];
  s = ss[0][r];
  for (int i = 1; i < 32; ++i) merge(m, s, sm[i][r], ss[i][r]);  // every thread of a row, in the same order
  const float log_s = log2f(s);
  if (p) {
    float sum = 0.f;
    if (pos < rows) {
      const size_t row = (size_t)rowmap[pos] * k;
      for (int i = slice; i < k; i += 32) {
        const float q = p[row + i], z = zk[(size_t)pos * k + i];
        if (q > 0.f) sum += q * (logf(q) - LN2 * (__builtin_fmaf(z, sc, -m) - log_s));
        else if (q != q || z != z) sum = NAN;
      }
    }
    sd[slice][r] = sum;
    __syncthreads();
  }
  if (threadIdx.x < 8 && pos < rows) {
    float sum = 0.f;
    if (p) {
      for (int i = 0; i < 32; ++i) sum += sd[i][r];
    } else {
      sum = LN2 * (log_s - __builtin_fmaf(zk[pos], sc, -m));
    }
    const float out = t2 * sum;
    lse[pos] = m + log_s;
    __hip_atomic_store(rowloss + pos, out, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (!reduction) loss[rowmap[pos]] = out;
  }
  if (!done) return;
  __shared__ int last;
  __shared__ double part_sum[4];
  __syncthreads();
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  double total = 0.;
  for (int i = threadIdx.x; i < rows; i += 256)
    total += __hip_atomic_load(rowloss + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o, 64);
  if ((threadIdx.x & 63) == 0) part_sum[threadIdx.x >> 6] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    total = part_sum[0] + part_sum[1] + part_sum[2] + part_sum[3];
    loss[0] = (float)(reduction == 2 ? total / max(rows, 1) : total);
  }
}

// The sum or mean of the rows' losses, in a fixed order.
__global__ __launch_bounds__(1024) void k_reduce(const float* __restrict__ rowloss, const int* __restrict__ count,
                                                 int reduction, float* __restrict__ loss) {
  __shared__ double sum[16];
  const int rows = count[0];
  double s = 0.;
#pragma unroll 8
  for (int i = threadIdx.x; i < rows; i += 1024) s += rowloss[i];
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) sum[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) s += sum[i];
    loss[0] = (float)(reduction == 2 ? s / max(rows, 1) : s);
  }
}

// fp16 without a reduction: factor[pos] = span g / max|g|, factor[n] = max|g| T / span, with the largest
// finite |g|, so that an infinite one (a loss scale that was too high) leaves the other tokens theirs.
__global__ __launch_bounds__(1024) void k_factor(const float* __restrict__ grad, long long ldg,
                                                 const int* __restrict__ rowmap, const int* __restrict__ count, int n,
                                                 float t, float span, float* __restrict__ factor) {
  __shared__ float top[16];
  const int rows = count[0];
  float m = 0.f;
#pragma unroll 8
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float g = fabsf(grad[rowmap[i] * ldg]);
    m = g < INFINITY ? fmaxf(m, g) : m;
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();
  for (int i = 0; i < 16; ++i) m = fmaxf(m, top[i]);
  if (m == 0.f) m = 1.f;
#pragma unroll 8
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float g = grad[rowmap[i] * ldg];
    factor[i] = g == 0.f ? 0.f : g / m * span;
  }
  if (threadIdx.x == 0) factor[n] = m * t / span;
}

// Puts a teacher's targets into the piece's dl: f (q - sum of the p of that id).  One wave a row,
// whose lanes compare their entries with 4 of the list at a time (30 x 127: 20 us one at a time, 11 us).
// The first RESIDUALS entries of the list whose derivative is large are those that are made good.
template <bool F16>
__global__ __launch_bounds__(256) void k_fix(const long long* __restrict__ ids, const float* __restrict__ p, int k,
                                             long long v, const float* __restrict__ zk, const float* __restrict__ lse,
                                             Upstream<F16> up, float sc, long long v0, long long vn,
                                             void* __restrict__ dl, long long lddl, int* __restrict__ at,
                                             float* __restrict__ lost, void* __restrict__ low) {
  using T = typename Type<F16>::T;
  __shared__ __attribute__((aligned(16))) int list[4][MAX_TARGETS];  // vocabulary entries, -1: none
  __shared__ __attribute__((aligned(16))) float prob[4][MAX_TARGETS];
  const int wave = threadIdx.x >> 6, pos = blockIdx.x * 4 + wave, lane = threadIdx.x & 63;
  if (pos >= up.count[0]) return;
  const size_t row = (size_t)up.rowmap[pos] * k;
  const int k4 = (k + 3) & ~3;
  for (int i = lane; i < k4; i += 64) {
    const long long id = i < k ? ids[row + i] : -1;
    list[wave][i] = id >= 0 && id < v ? (int)id : -1;
    prob[wave][i] = i < k ? p[row + i] : 0.f;
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own list: no barrier
  const float f = up.of(pos), ls = lse[pos];
  int large = 0;
  for (int i0 = 0; i0 < k; i0 += 64) {
    const int i = i0 + lane, id = i < k ? list[wave][i] : -1;
    float sum = 0.f;
    bool firstone = id >= 0;
#pragma unroll 4
    for (int o = 0; o < k4; o += 4) {
      const u32x4 other = *reinterpret_cast<const u32x4*>(&list[wave][o]);
      const f32x4 q = *reinterpret_cast<const f32x4*>(&prob[wave][o]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool same = (int)other[e] == id;
        sum += same ? q[e] : 0.f;
        firstone &= !same || o + e >= i;
      }
    }
    const float g = firstone ? __builtin_amdgcn_exp2f(zk[(size_t)pos * k + i] * sc - ls) - sum : 0.f;
    const unsigned long long mask = __ballot(fabsf(g) >= LARGE);
    const int slot = large + __popcll(mask & ((1ull << lane) - 1));
    large += __popcll(mask);
    if (!firstone) continue;
    const bool here = id >= v0 && id < v0 + vn;
    const T r = (T)(f * g);
    if (here) static_cast<T*>(dl)[(size_t)pos * lddl + (id - v0)] = r;
    if (here && low) static_cast<T*>(low)[(size_t)pos * lddl + (id - v0)] = (T)(f * g - (float)r);
    if (fabsf(g) >= LARGE && slot < RESIDUALS) {
      if (v0 == 0) at[pos * RESIDUALS + slot] = id;
      if (here) lost[pos * RESIDUALS + slot] = f * g - (float)r;
    }
  }
  if (v0 == 0 && lane >= large && lane < RESIDUALS) at[pos * RESIDUALS + lane] = -1;
}

// Joins the splits of dX, adds what dl's rounding took, scales, rounds once, and puts zeros into
// the rows without a loss.
template <bool F16>
__global__ __launch_bounds__(256) void k_dx_out(const float* __restrict__ part, const int* __restrict__ chosen, int d, int dp,
                                                const int* __restrict__ posof, Upstream<F16> up,
                                                const int* __restrict__ at, const float* __restrict__ lost,
                                                int residuals, const void* __restrict__ w, long long ldw,
                                                void* __restrict__ dx) {
  using T = typename Type<F16>::T;
  typedef __attribute__((ext_vector_type(4))) T t4;
  const int per_row = (d + 1023) / 1024, row = blockIdx.x / per_row, pos = posof[row];
  const int c = ((blockIdx.x - row * per_row) * 256 + threadIdx.x) * 4;
  if (c >= d) return;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (pos >= 0) {
    const int rows = up.count[0], splits = *chosen;
    const float* from = part + (size_t)pos * dp + c;
    int i = 0;
    for (; i + 8 <= splits; i += 8) {  // 8 loads in flight, added in order
      f32x4 v[8];
#pragma unroll
      for (int o = 0; o < 8; ++o) v[o] = *reinterpret_cast<const f32x4*>(from + (size_t)(i + o) * rows * dp);
#pragma unroll
      for (int o = 0; o < 8; ++o) s += v[o];
    }
    for (; i < splits; ++i) s += *reinterpret_cast<const f32x4*>(from + (size_t)i * rows * dp);
    for (int r = 0; r < residuals; ++r) {
      const int id = at[pos * residuals + r];
      if (id < 0) break;
      const t4 v = *reinterpret_cast<const t4*>(static_cast<const T*>(w) + id * ldw + c);
      const float l = lost[pos * residuals + r];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += l * (float)v[e];
    }
    s *= up.scale();
  }
  T* out = static_cast<T*>(dx) + (size_t)row * d + c;
  if (c + 4 <= d) {
    const u32x2 v = {pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3])};
    __builtin_memcpy(out, &v, 8);  // at any alignment
  } else {
    for (int e = 0; e < 4 && c + e < d; ++e) out[e] = (T)s[e];
  }
}

int padded(long long d) { return (int)((d + 63) / 64 * 64); }

int residuals(const tkl_args& a) { return a.distill ? RESIDUALS : 1; }
int halves(const tkl_args& a) { return a.small & 8 ? 2 : 1; }  // parts of dl

// What the forward pass keeps, in one buffer.  Without a teacher p and flag are not there.
struct Kept {
  char* xc;                        // [n][dp], the packed rows
  float *lse, *rowloss;            // by packed row
  int *rowmap, *posof, *count;     // packed row -> token and back; count[0] packed rows, count[1] k_loss's
  float *zk, *p;                   // [packed row][k] logits of the targets; a teacher's [token][k] probabilities
  int* flag;                       // by token: whether it has a target
  int* at;                         // [packed row][residuals] vocabulary entries, -1: none
  long long bytes;
};
Kept kept_of(const tkl_args& a) {
  Kept r;
  const long long n = a.n, lists = a.distill ? n * a.k : 0;
  char* at = static_cast<char*>(a.kept);
  auto take = [&](long long size) {
    char* was = at;
    at += size;
    return was;
  };
  r.xc = take(2 * n * padded(a.d));
  r.lse = reinterpret_cast<float*>(take(4 * n));
  r.rowloss = reinterpret_cast<float*>(take(4 * n));
  r.rowmap = reinterpret_cast<int*>(take(4 * n));
  r.posof = reinterpret_cast<int*>(take(4 * n));
  r.count = reinterpret_cast<int*>(take(8));
  r.zk = reinterpret_cast<float*>(take(4 * (a.distill ? lists : n)));
  r.p = a.distill ? reinterpret_cast<float*>(take(4 * lists)) : nullptr;
  r.flag = a.distill ? reinterpret_cast<int*>(take(4 * n)) : nullptr;
  r.at = reinterpret_cast<int*>(take(4 * n * residuals(a)));
  r.bytes = at - static_cast<char*>(a.kept);
  return r;
}
// The backward pass' workspace, in one buffer.
struct Room {
  void* dl;       // [n][piece] 16-bit
  void* low;      // the same, what dl's rounding took, or null
  float* sums;    // [splits][packed rows][dp] of dX: n dp, or what `fill` tiles hold
  float* factor;  // [n + 1]
  int* splits;    // of dX, as k_dx found them
  float* lost;    // [packed row][residuals] what dl's rounding took
  int *listed, *starts;  // k_list's, of more than FEW_ROWS tokens: [packed row][residuals], [piece / BUCKET + 1]
  float* parts;   // [parts][v][dp] of dW, where there are more than one
  void* xt;       // Xc^T [dp][n up to 64], for dW in large tiles
  long long bytes;
};
Room room_of(const tkl_args& a) {
  Room r;
  char* at = static_cast<char*>(a.room);
  r.dl = at;
  r.low = halves(a) > 1 ? at + 2 * a.n * a.piece : nullptr;
  at += 2 * a.n * a.piece * halves(a);
  r.sums = reinterpret_cast<float*>(at);
  const long long once = a.n * padded(a.d), tile = a.small & 2 ? Small::BM * Small::BN : Big::BM * Big::BN;
  if (a.want & 1) at += 4 * std::max(once, std::min(a.piece / 512 * once, a.fill * tile));
  r.factor = reinterpret_cast<float*>(at);
  at += 4 * (a.n + 1);
  r.splits = reinterpret_cast<int*>(at);
  at += 4;
  r.lost = reinterpret_cast<float*>(at);
  at += 4 * a.n * residuals(a);
  r.listed = r.starts = nullptr;
  if ((a.want & 2) && halves(a) == 1 && a.n > FEW_ROWS) {
    r.listed = reinterpret_cast<int*>(at);
    at += 4 * a.n * residuals(a);
    r.starts = reinterpret_cast<int*>(at);
    at += 4 * (a.piece / BUCKET + 1);
  }
  at += -(at - static_cast<char*>(a.room)) & 15;
  r.parts = reinterpret_cast<float*>(at);
  if (a.parts > 1) at += 4 * a.parts * a.v * padded(a.d);
  r.xt = at;
  if ((a.want & 2) && !(a.small & 4)) at += 2 * padded(a.d) * (long long)padded(a.n);
  r.bytes = at - static_cast<char*>(a.room);
  return r;
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

int check(const tkl_args& a) {
  const char* bad = nullptr;
  if (a.n < 1 || a.n > (1 << 20)) bad = "tokens must be 1 to 2^20";
  else if (a.d < 1 || a.d > (1 << 16)) bad = "the width must be 1 to 65536";
  else if (a.v < 1 || a.v > (1 << 24)) bad = "the vocabulary must have 1 to 2^24 entries";
  else if (a.k < 1 || a.k > MAX_TARGETS) bad = "1 to 1024 targets a token";
  else if (!a.wc && ((a.d & 7) || (a.ldw & 7) || (reinterpret_cast<uintptr_t>(a.w) & 15)))
    bad = "w's rows are not 16-byte aligned and there is no room for a copy";
  else if (!a.wc && (a.ldw < a.d || a.ldw > (1 << 21))) bad = "w's row stride must be its width to 2^21 elements";
  // a launch has fewer than 2^32 threads: 512 to a tile of 256 x 256, 256 to 1024 numbers of dX
  else if ((a.v + 255) / 256 * ((a.n + 255) / 256) >= 1 << 23) bad = "tokens x vocabulary must be below 2^39";
  else if ((a.d + 1023) / 1024 * a.n >= 1 << 24) bad = "tokens x width must be below 2^34";
  else if (a.reduction < 0 || a.reduction > 2) bad = "reduction must be 0 to 2";
  else if (!(a.temperature >= 0x1p-32f && a.temperature <= 0x1p32f)) bad = "the temperature must be 2^-32 to 2^32";
  if (bad) {
    snprintf(g_err, sizeof(g_err), "%s", bad);
    return -1;
  }
  return 0;
}

// A matrix product's kernel may use more LDS than the default limit.
template <class Kernel>
hipError_t allow(Kernel* k, int lds) {
  return hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
}
template <class Tile, bool F16>
hipError_t allow_all() {
  hipError_t e = allow(&k_logits<Tile, F16, LSE>, Tile::LDS);
  if (e == hipSuccess) e = allow(&k_logits<Tile, F16, DL>, Tile::LDS);
  if (e == hipSuccess) e = allow(&k_logits<Tile, F16, TWO>, Tile::LDS);
  if (e == hipSuccess) e = allow(&k_logits<Tile, F16, KEEP>, Tile::LDS);
  if (e == hipSuccess) e = allow(&k_dx<Tile, F16>, Tile::LDS);
  if (e == hipSuccess) e = allow(&k_dw<Tile, F16, false>, Tile::LDS);
  if (e == hipSuccess) e = allow(&k_dw<Tile, F16, true>, Tile::LDS);
  return e;
}
hipError_t set_lds_limit() {
  static std::once_flag once[64];
  static hipError_t result[64];
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
  std::call_once(once[dev], [dev] {
    result[dev] = allow_all<Big, false>();
    if (result[dev] == hipSuccess) result[dev] = allow_all<Big, true>();
    if (result[dev] == hipSuccess) result[dev] = allow_all<Small, false>();
    if (result[dev] == hipSuccess) result[dev] = allow_all<Small, true>();
  });
  return result[dev];
}

unsigned blocks(long long items, long long per) { return (unsigned)((items + per - 1) / per); }

template <typename T>
void pad(const tkl_args& a, int dp, hipStream_t s) {
  if (a.wc)
    k_pad<T><<<(unsigned)std::min<long long>(blocks(a.v * (dp / 8), 256), 16384), 256, 0, s>>>(
        static_cast<const T*>(a.w), a.ldw, a.v, (int)a.d, dp, static_cast<T*>(a.wc));
}

// Where the forward pass puts the tiles' maxima and sums: behind the codes, if they are kept.
float2* part_of(const tkl_args& a) {
  return reinterpret_cast<float2*>(a.codes ? static_cast<char*>(a.codes) + 2 * a.n * Codes::stride(a.v)
                                           : static_cast<char*>(a.room));
}

template <class Tile, bool F16, Mode MODE>
void logits_as(const tkl_args& a, const Kept& kept, const Weight& w, int dp, long long v0, int vn, const Upstream<F16>& up,
               void* out, long long ldout, float* of_target, void* low, hipStream_t s) {
  k_logits<Tile, F16, MODE><<<blocks(vn, Tile::BM) * blocks(a.n, Tile::BN), Tile::THREADS, Tile::LDS, s>>>(
      w.at, w.ldb, kept.xc, (long long)dp * 2, (int)v0, (int)v0 + vn, w.dk, kept.count, (int)a.n, LOG2E / a.temperature,
      part_of(a), kept.lse, up, a.distill ? nullptr : kept.at, out, ldout, of_target, low);
}

template <class Tile, bool F16>
void all_logits(const tkl_args& a, const Kept& q, const Weight& w, int dp, hipStream_t s) {
  if (a.codes) logits_as<Tile, F16, KEEP>(a, q, w, dp, 0, (int)a.v, {}, a.codes, Codes::stride(a.v), q.zk, nullptr, s);
  else logits_as<Tile, F16, LSE>(a, q, w, dp, 0, (int)a.v, {}, nullptr, 0, q.zk, nullptr, s);
}

// dl of a piece, out of the kept logits or by computing them again
template <class Tile, bool F16>
void derivative(const tkl_args& a, const Kept& q, const Weight& w, int dp, long long v0, int vn, const Upstream<F16>& up,
                const Room& r, hipStream_t s) {
  if (a.codes)
    k_dl<Tile, F16><<<blocks(a.piece, 2048) * (unsigned)a.n, 256, 0, s>>>(
        static_cast<const unsigned short*>(a.codes), Codes::stride(a.v), part_of(a), (int)a.n, (int)v0, vn,
        LOG2E / a.temperature, q.lse, up, a.distill ? nullptr : q.at, q.zk, r.dl, a.piece, r.lost);
  else if (r.low)
    logits_as<Tile, F16, TWO>(a, q, w, dp, v0, vn, up, r.dl, a.piece, r.lost, r.low, s);
  else
    logits_as<Tile, F16, DL>(a, q, w, dp, v0, vn, up, r.dl, a.piece, r.lost, nullptr, s);
}

template <bool F16>
hipError_t forward(const tkl_args& a) {
  using T = typename Type<F16>::T;
  hipStream_t s = static_cast<hipStream_t>(a.stream);
  const int n = (int)a.n, d = (int)a.d, k = (int)a.k, dp = padded(a.d);
  const long long* ids = static_cast<const long long*>(a.ids);
  const Kept q = kept_of(a);
  float *loss = static_cast<float*>(a.loss), t = a.temperature;
  T* xc = reinterpret_cast<T*>(q.xc);
  if (a.distill)
    k_teacher<<<blocks(n, 4), 256, 0, s>>>(ids, static_cast<const float*>(a.teacher), n, k, 1.f / t, q.p, q.flag);
  const int per = gather_rows(n);
  k_gather<T><<<blocks(n, 4 * per), 256, 0, s>>>(static_cast<const T*>(a.x), a.ldx, n, d, dp, ids, a.ignore, q.flag, xc,
                                                 q.rowmap, q.posof, q.count, a.reduction ? nullptr : loss, per, a.v, q.at,
                                                 q.zk);
  pad<T>(a, dp, s);
  const Weight w = weight_of(a, dp);
  if (a.small & 1) all_logits<Small, F16>(a, q, w, dp, s);
  else all_logits<Big, F16>(a, q, w, dp, s);
  if (a.distill)
    k_dots<F16><<<(unsigned)std::min<long long>((n * ((k + 15ll) / 16) + 3) / 4, 1 << 22), 256, 0, s>>>(
        xc, dp, w.at, w.ldb / 2, w.dk, ids, k, a.v, q.rowmap, q.count, q.zk);
  k_loss<<<blocks(n, 8), 256, 0, s>>>(part_of(a), (int)blocks(a.v, a.small & 1 ? Small::BM : Big::BM), n, q.zk, q.p, k,
                                      q.rowmap, q.count, LOG2E / t, t * t, q.lse, q.rowloss, loss, a.reduction,
                                      a.reduction && n <= 512 ? q.count + 1 : nullptr);
  if (a.reduction && n > 512) k_reduce<<<1, 1024, 0, s>>>(q.rowloss, q.count, a.reduction, loss);
  return hipGetLastError();
}

template <class Tile, bool F16>
void dx(const tkl_args& a, const Kept& q, const Room& r, const Weight& w, int dp, long long v0, int vn, hipStream_t s) {
  const unsigned most = std::max<long long>((long long)blocks(w.dk, Tile::BM) * blocks(a.n, Tile::BN), a.fill);
  k_dx<Tile, F16><<<most, Tile::THREADS, Tile::LDS, s>>>(w.at, w.ldb, r.dl, a.piece * 2, (int)v0, vn, w.dk, dp, q.count,
                                                         (int)a.fill, v0 == 0, r.sums, r.splits);
  if (r.low)
    k_dx<Tile, F16><<<most, Tile::THREADS, Tile::LDS, s>>>(w.at, w.ldb, r.low, a.piece * 2, (int)v0, vn, w.dk, dp,
                                                           q.count, (int)a.fill, 0, r.sums, r.splits);
}

template <class Tile, bool F16>
void dw(const tkl_args& a, const Kept& q, const Room& r, int dp, long long v0, int vn, const Upstream<F16>& up,
        hipStream_t s) {
  const dim3 grid(blocks(a.d, Tile::BM) * blocks(vn, Tile::BN), std::max(1, a.parts));
  if (r.listed)
    k_list<<<blocks(vn, BUCKET), 1024, 0, s>>>(q.at, residuals(a), q.count, (int)v0, vn, r.listed, r.starts);
  auto* kernel = r.low ? &k_dw<Tile, F16, true> : &k_dw<Tile, F16, false>;
  kernel<<<grid, Tile::THREADS, Tile::LDS, s>>>(r.xt, 2 * padded(a.n), q.xc, dp, r.dl, a.piece * 2, (int)v0, vn, (int)a.d,
                                                q.count, up, q.at, r.lost, residuals(a), a.dw, (int)a.d, r.parts, r.low, r.listed,
                                                r.starts);
  if (a.parts > 1)
    k_dw_out<F16><<<blocks(a.v * (dp / 4), 256), 256, 0, s>>>(r.parts, a.parts, a.v, (int)a.d, dp, up, a.dw);
}

template <bool F16>
hipError_t backward(const tkl_args& a) {
  hipStream_t s = static_cast<hipStream_t>(a.stream);
  const int n = (int)a.n, d = (int)a.d, k = (int)a.k, dp = padded(a.d);
  const Kept q = kept_of(a);
  const Room r = room_of(a);
  const Upstream<F16> up = {static_cast<const float*>(a.grad), q.rowloss, r.factor, q.rowmap, q.count, a.ldg, a.reduction,
                            n, a.temperature};
  if (F16 && a.reduction == 0)
    k_factor<<<1, 1024, 0, s>>>(up.grad, up.ldg, up.rowmap, up.count, n, a.temperature, Upstream<F16>::SPAN, r.factor);
  using T = typename Type<F16>::T;
  if ((a.want & 2) && !(a.small & 4))
    k_transpose<T><<<dim3(dp / 64, blocks(n, 64)), 256, 0, s>>>(reinterpret_cast<const T*>(q.xc), dp, q.count,
                                                                static_cast<T*>(r.xt), padded(n));
  const Weight w = weight_of(a, dp);
  for (long long v0 = 0; v0 < a.v; v0 += a.piece) {
    const int vn = (int)std::min(a.piece, a.v - v0);
    if (a.small & 1) derivative<Small, F16>(a, q, w, dp, v0, vn, up, r, s);
    else derivative<Big, F16>(a, q, w, dp, v0, vn, up, r, s);
    if (a.distill)
      k_fix<F16><<<blocks(n, 4), 256, 0, s>>>(static_cast<const long long*>(a.ids), q.p, k, a.v, q.zk, q.lse, up,
                                              LOG2E / a.temperature, v0, vn, r.dl, a.piece, q.at, r.lost, r.low);
    if (a.want & 1) {
      if (a.small & 2) dx<Small, F16>(a, q, r, w, dp, v0, vn, s);
      else dx<Big, F16>(a, q, r, w, dp, v0, vn, s);
    }
    if (a.want & 2) {
      if (a.small & 4) dw<Small, F16>(a, q, r, dp, v0, vn, up, s);
      else dw<Big, F16>(a, q, r, dp, v0, vn, up, s);
    }
  }
  if (a.want & 1)
    k_dx_out<F16><<<blocks(d, 1024) * (unsigned)n, 256, 0, s>>>(r.sums, r.splits, d, dp, q.posof, up, q.at, r.lost,
                                                                r.low ? 0 : residuals(a), w.at, w.ldb / 2, a.dx);
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

// What the caller has to agree on: the struct's size, and the bytes of its `kept` and (with a
// piece) backward's `room`.
extern "C" int tkl_args_size() { return (int)sizeof(tkl_args); }
extern "C" long long tkl_kept_bytes(const tkl_args* a) { return kept_of(*a).bytes; }
extern "C" long long tkl_room_bytes(const tkl_args* a) { return room_of(*a).bytes; }

// Both are queued on a->stream and wait for nothing.  0, or -1 / a HIP error (tkl_last_error).
extern "C" int tkl_forward(const tkl_args* a) { return on_device(a, a->f16 ? forward<true> : forward<false>); }

extern "C" int tkl_backward(const tkl_args* a) {
  if (a->parts < 0 || a->parts > 64 || (a->parts > 1 && a->piece < a->v)) {
    snprintf(g_err, sizeof(g_err), "dW in %d parts: at most 64, of one piece", a->parts);
    return -1;
  }
  if (halves(*a) > 1 && a->codes) {
    snprintf(g_err, sizeof(g_err), "kept logits are rounded: their derivative has no second part");
    return -1;
  }
  // (a tile's rows of dl are addressed below FAR)
  if (a->piece < Big::BM || a->piece % Big::BM || a->piece > (1 << 24) || a->fill < 1 || a->fill > 4096 ||
      std::min<long long>(a->n, Big::BN) * a->piece >= (1 << 29)) {
    snprintf(g_err, sizeof(g_err), "piece %lld must be a multiple of %d, below 2^29 over 256 tokens; fill %lld 1 to 4096",
             a->piece, Big::BM, a->fill);
    return -1;
  }
  // dX in large tiles: the copies of a tile start at its rows 0, 64, 128 and 192, which are known not to
  // be there by how far behind the last one they lie, in 32 bits with a sign
  if ((a->want & 1) && !(a->small & 2) && (193 - std::min<long long>(a->n, 193)) * 2 * a->piece >= (1ll << 31)) {
    snprintf(g_err, sizeof(g_err), "rows of %lld entries are too long for %lld tokens in large tiles", a->piece, a->n);
    return -1;
  }
  return on_device(a, a->f16 ? backward<true> : backward<false>);
}
