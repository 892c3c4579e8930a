// Matrix-vector products with 4-bit weights on MI355X (gfx950): y = x W^T for 1 to 64 rows of
// x, W[n][k] = scale[n][k/group] (code[n][k] - zero[n][k/group]).
//
// A product of so few rows reads each weight once and is bound by that read, so the codes
// stay packed until they are in registers.  A code c becomes the 16-bit number 16 + c by bit
// operations alone (its 4 bits are the top of the mantissa of a number in [16, 32), exact in
// bf16 and fp16), the matrix cores sum (16 + c) x in fp32, and per group
//
//     scale (sum (16 + c) x - (16 + zero) sum x)
//
// is added to the result in fp32; sum x comes from one more matrix instruction with ones.
// Nothing is rounded to 16 bits on the way but the result.
//
// Measured (device time, weights in turn, so out of HBM): one row, 131072 x 4096 with groups of 64
// and zeros, 60 us, 4.9 TB/s; 8192 x 8192 11.2 us; 64 rows, 16384 x 16384 58 us and 6 to join.
// One row is bound by the reads and the instructions that unpack and scale; many rows by the vector
// and the matrix instructions, 23 and 14 us, which hardly overlap (42 us without loads, barriers
// and x's way through LDS, 54 without the loads, 49 with nothing but loads).
//
// C ABI for ctypes: triton_kubernetes_amd/ops/gemv.py.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;

static thread_local char g_err[512];

extern "C" const char* tkv_last_error() { return g_err; }

namespace {

template <bool F16>
struct Type;
template <>
struct Type<false> {
  using T = __bf16;
  static constexpr unsigned MASK = 0x00780078u, SIXTEEN = 0x41804180u, ONES = 0x3f803f80u;  // mantissa bits 3-6
  static constexpr int LOW = 3;
  static __device__ __forceinline__ float sum2(unsigned v, float c) {  // c + both numbers
    typedef __attribute__((ext_vector_type(2))) __bf16 t2;
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(t2, v), __builtin_bit_cast(t2, ONES), c, false);
  }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
};
template <>
struct Type<true> {
  using T = _Float16;
  static constexpr unsigned MASK = 0x03c003c0u, SIXTEEN = 0x4c004c00u, ONES = 0x3c003c00u;  // mantissa bits 6-9
  static constexpr int LOW = 6;
  static __device__ __forceinline__ float sum2(unsigned v, float c) {
    typedef __attribute__((ext_vector_type(2))) _Float16 t2;
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(t2, v), __builtin_bit_cast(t2, ONES), c, false);
  }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
};

// The 8 codes of a dword as 16 + c, in the order (0,4) (1,5) (2,6) (3,7): one shift and one
// and-or a pair.
template <bool F16>
__device__ __forceinline__ u32x4 unpack(unsigned w) {
  using Y = Type<F16>;
  u32x4 r;
  unsigned mask = Y::MASK, sixteen = Y::SIXTEEN;
  asm("" : "+s"(mask), "+v"(sixteen));  // in registers, or the and-or becomes two instructions
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int up = Y::LOW - 4 * i;
    const unsigned s = up >= 0 ? w << (up & 31) : w >> (-up & 31);
    r[i] = (s & mask) | sixteen;
  }
  return r;
}

// 8 numbers of x in the order that unpack gives the codes
__device__ __forceinline__ u32x4 pairs(u32x4 v) {
  return u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
               __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// 4x4 transpose between the dwords of a lane and the four 16-lane rows of a wave: afterwards
// dword s of row j is what dword j of row s was.
__device__ __forceinline__ u32x4 exchange(u32x4 d) {
  const auto a = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto e = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4{c[0], c[1], e[0], e[1]};
}

constexpr int CHUNK = 128;  // columns: 16 bytes of codes for each of the 4 lanes of a row

// The scales and zeros of one row and chunk, as they were loaded, so that nothing waits for them
// before their use.  G: scales of a chunk, 1, 2 or 4 for groups of whole chunks, of 64 and of
// 32; 0 for any other group: 4, each column block of 32 with the scale of whatever group it is in.
template <bool F16, int G, bool ZEROS>
struct Scales {
  using T = typename Type<F16>::T;
  static constexpr int SPC = G ? G : 4, NS = G ? (SPC + 1) / 2 : SPC, NZ = G ? 1 : SPC;
  static constexpr int LOADS = (G ? 1 : SPC) * (ZEROS ? 2 : 1);
  unsigned s[NS], z[NZ];

  static __device__ __forceinline__ Scales load(const T* s_row, const uint8_t* z_row, int chunk, int groups,
                                                int per_group, int group, int k) {
    Scales f = {};
    if constexpr (G == 1) {
      const int g = per_group == 1 ? chunk : chunk / per_group;
      uint16_t v;
      __builtin_memcpy(&v, s_row + g, 2);
      f.s[0] = v;
      if constexpr (ZEROS) f.z[0] = z_row[g];
    } else if constexpr (G) {
      const int g = min(chunk * SPC, groups - SPC);  // the last chunk may have fewer: of() shifts
      __builtin_memcpy(f.s, s_row + g, 2 * SPC);
      if constexpr (ZEROS && G == 2) {
        uint16_t v;
        __builtin_memcpy(&v, z_row + g, 2);
        f.z[0] = v;
      } else if constexpr (ZEROS) {
        __builtin_memcpy(f.z, z_row + g, 4);
      }
    } else {
#pragma unroll
      for (int q = 0; q < SPC; ++q) {
        const int g = min(chunk * CHUNK + q * 32, k - 1) / group;
        uint16_t v;
        __builtin_memcpy(&v, s_row + g, 2);
        f.s[q] = v;
        if constexpr (ZEROS) f.z[q] = z_row[g];
      }
    }
    return f;
  }
  // those that lane from / 4 loaded, which are of chunk `chunk`
  __device__ __forceinline__ Scales of(int from, int chunk, int groups) const {
    Scales v;
#pragma unroll
    for (int i = 0; i < NS; ++i) v.s[i] = __builtin_amdgcn_ds_bpermute(from, s[i]);
    if constexpr (ZEROS) {
#pragma unroll
      for (int i = 0; i < NZ; ++i) v.z[i] = __builtin_amdgcn_ds_bpermute(from, z[i]);
    }
    if constexpr (G > 1) {
      const int gone = chunk * SPC + SPC - groups;
      if (gone > 0) {  // the scales that are not there become 0
        if constexpr (G == 2) {
          v.s[0] >>= 16;
        } else {
          const uint64_t t = ((uint64_t)v.s[1] << 32 | v.s[0]) >> (16 * gone);
          v.s[0] = (unsigned)t;
          v.s[1] = (unsigned)(t >> 32);
        }
        if constexpr (ZEROS) v.z[0] >>= 8 * gone;
      }
    }
    return v;
  }
  __device__ __forceinline__ float scale(int q) const {
    return (float)__builtin_bit_cast(T, (uint16_t)(G ? s[q / 2] >> (q % 2 * 16) : s[q]));
  }
  static constexpr float OFFSET = 16.f + 8.f;             // without zeros
  __device__ __forceinline__ float offset(int q) const {  // of the number that a code of zero unpacks to
    return ZEROS ? 16.f + (float)(G ? z[0] >> (q * 8) & 255 : z[q]) : OFFSET;
  }
};

// One row of x (blockIdx.y).  WN tiles of 16 rows of W a workgroup, WK waves to a tile, which
// share its columns.
//
// The codes go to LDS by copies without registers, a stage of 16 rows x 256 bytes (4 chunks of
// 128 columns) at a time and wave, two stages in flight: 16 neighbouring lanes read 256 bytes of
// one row.  (Loading them straight to where the matrix cores want them, neighbouring lanes in
// different rows, took 120 us instead of 71 us for 131072 x 4096: every lane was a cache line of
// its own to look up.)  Unit u of row r lies at u ^ r, so the reads conflict on no banks.
// Scales and zeros: lane (j, r) loads those of row r and chunk j of the stage, and the others
// get them from it.
//
// x goes through LDS a segment of `seg` chunks at a time, in the order that the codes unpack
// to.  Columns behind k are zeros in x, so whatever codes are read there change nothing.  All 16
// rows of the matrix instruction get the same x; the first one's sums are kept.
//
// The waits count what is in flight, so no load may move across the empty asm statements: the
// pointers are not __restrict__, which would let the compiler do that.
constexpr int STAGE = 4, STAGES = 2, STAGE_BYTES = 16 * STAGE * CHUNK / 2, SEGMENT = 256;

template <bool F16, int G, bool ZEROS, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK) void k_one(const void* xs_in, long long ldx, const uint8_t* codes,
                                                      const void* scales, const uint8_t* zeros, void* y, long long ldy,
                                                      int n, int k, int group, int seg) {
  using Y = Type<F16>;
  using T = typename Y::T;
  using Sc = Scales<F16, G, ZEROS>;
  constexpr int STEPS = 4 / Sc::SPC, THREADS = 64 * WN * WK;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  u32x4* xs = reinterpret_cast<u32x4*>(smem + WN * WK * STAGES * STAGE_BYTES);
  const T* x = static_cast<const T*>(xs_in) + blockIdx.y * ldx;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave % WK, wn = wave / WK, j = lane >> 4, r = lane & 15;
  const int row0 = (blockIdx.x * WN + wn) * 16, row = row0 + r, groups = k / group, per_group = group / CHUNK;
  const int chunks = (k + CHUNK - 1) / CHUNK;
  char* mine = smem + wave * STAGES * STAGE_BYTES;
  // rows past n and columns past the last row's end read as zeros
  const uint64_t at0 = reinterpret_cast<uint64_t>(codes) + (uint64_t)min(row0, n - 1) * (k / 2);
  const uint64_t base = (uint64_t)__builtin_amdgcn_readfirstlane((unsigned)(at0 >> 32)) << 32 |
                        (unsigned)__builtin_amdgcn_readfirstlane((unsigned)at0);
  const auto buffer = __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void*>(base), 0, __builtin_amdgcn_readfirstlane(max(0, min(16, n - row0)) * (k / 2)), 0x00020000);
  const int safe = min(row, n - 1);
  const T* s_row = static_cast<const T*>(scales) + (size_t)safe * groups;
  const uint8_t* z_row = ZEROS ? zeros + (size_t)safe * groups : nullptr;
  constexpr int LOADS = 4 + Sc::LOADS;  // of copy() and fetch()

  int off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) off[i] = (i * 4 + j) * (k / 2) + ((r ^ (i * 4 + j)) * 16);
  // the codes of chunks c .. c + 3, of nothing past `end`
  auto copy = [&](int c, int end, int slot) {
    const int at = c < end ? c * (CHUNK / 2) : 0x40000000;  // (a row's codes are at most 2^19 bytes)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          buffer, (__attribute__((address_space(3))) void*)(mine + slot * STAGE_BYTES + i * 1024), 16, off[i] + at, 0, 0,
          0);
  };
  auto fetch = [&](int c) { return Sc::load(s_row, z_row, min(c + j, chunks - 1), groups, per_group, group, k); };
  float total = 0.f;
  const u32x4 ones = {Y::ONES, Y::ONES, Y::ONES, Y::ONES};
  const int lane_at = r * 256 + r * 16 + j * 4;
  // chunk u of the stage, chunk c of the segment, chunk `all` of the row
  auto add = [&](const Sc& f, const char* img, int u, int c, int all) {
    const Sc v = f.of((u * 16 + r) * 4, all, groups);
    f32x4 part = {0.f, 0.f, 0.f, 0.f}, sum = part;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const unsigned w = *reinterpret_cast<const unsigned*>(img + (lane_at ^ ((u * 4 + s) * 16)));
      const u32x4 a = xs[c * 16 + s * 4 + j];
      part = Y::mfma(a, unpack<F16>(w), part);
      sum = Y::mfma(a, ones, sum);
      if ((s + 1) % STEPS == 0) {
        const int q = s / STEPS;
        total += v.scale(q) * (part[0] - v.offset(q) * sum[0]);
        part = sum = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  };

  for (int first = 0; first < chunks; first += seg) {
    const int here = min(seg, chunks - first), per = (here + WK - 1) / WK;
    const int c0 = wk * per, c1 = min(here, c0 + per);
    Sc f[STAGES];  // the first stages fly while x is brought in
#pragma unroll
    for (int t = 0; t < STAGES; ++t) {
      copy(first + c0 + t * STAGE, first + c1, t);
      f[t] = fetch(first + c0 + t * STAGE);
      asm volatile("" ::: "memory");  // in this order
    }
    if (first) __syncthreads();
    const int units = here * 16;
    for (int u0 = tid; u0 < units; u0 += THREADS * 4) {
      u32x4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int unit = u0 + i * THREADS, ks = first * CHUNK + unit * 8;
        v[i] = u32x4{0, 0, 0, 0};
        if (unit < units && ks < k) v[i] = *reinterpret_cast<const u32x4*>(x + ks);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (u0 + i * THREADS < units) xs[u0 + i * THREADS] = pairs(v[i]);
    }
    __syncthreads();
    for (int c = c0; c < c1; c += STAGE * STAGES) {
#pragma unroll
      for (int t = 0; t < STAGES; ++t) {
        const int at = c + t * STAGE;
        // loads return in order: of what is in flight, only the other stage's is younger
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * LOADS) : "memory");
        const Sc now = f[t];
        const char* img = mine + t * STAGE_BYTES;
        if (at + STAGE <= c1) {
          // all codes of the stage, and x one step ahead of the matrix instructions: left to
          // itself the compiler reads right before each use and waits every time
          unsigned w[STAGE * 4];
          u32x4 xa[2];
          const u32x4* x0 = xs + at * 16 + j;
#pragma unroll
          for (int i = 0; i < STAGE * 4; ++i) w[i] = *reinterpret_cast<const unsigned*>(img + (lane_at ^ (i * 16)));
          xa[0] = x0[0];
          Sc v[STAGE];
#pragma unroll
          for (int u = 0; u < STAGE; ++u) v[u] = now.of((u * 16 + r) * 4, first + at + u, groups);
          f32x4 part, sum;
#pragma unroll
          for (int i = 0; i < STAGE * 4; ++i) {
            if (i + 1 < STAGE * 4) xa[(i + 1) & 1] = x0[(i + 1) * 4];
            __builtin_amdgcn_sched_barrier(0);
            if (i % STEPS == 0) part = sum = f32x4{0.f, 0.f, 0.f, 0.f};
            part = Y::mfma(xa[i & 1], unpack<F16>(w[i]), part);
            sum = Y::mfma(xa[i & 1], ones, sum);
            if ((i + 1) % STEPS == 0) {
              const int q = i % 4 / STEPS;
              total += v[i / 4].scale(q) * (part[0] - v[i / 4].offset(q) * sum[0]);
            }
          }
        } else {
          for (int u = 0; at + u < c1; ++u) add(now, img, u, at + u, first + at + u);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read
        copy(first + at + STAGE * STAGES, first + c1, t);
        f[t] = fetch(first + at + STAGE * STAGES);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy lands in what LDS holds next
  }
  if constexpr (WK > 1) {
    float* sums = reinterpret_cast<float*>(smem);  // [wave][16]
    __syncthreads();
    if (j == 0) sums[wave * 16 + r] = total;
    __syncthreads();
    if (wk) return;
#pragma unroll
    for (int o = 1; o < WK; ++o) total += sums[(wave + o) * 16 + r];
  }
  if (j == 0 && row < n) static_cast<T*>(y)[blockIdx.y * ldy + row] = (T)total;
}

template <bool F16, int G, bool ZEROS, int WN, int WK>
hipError_t one_as(const void* x, long long ldx, const uint8_t* codes, const void* scales, const uint8_t* zeros, void* y,
                  long long ldy, int m, int n, int k, int group, hipStream_t s) {
  const int tiles = (n + 15) / 16, chunks = (k + CHUNK - 1) / CHUNK, seg = std::min(chunks, SEGMENT);
  const dim3 grid((tiles + WN - 1) / WN, m);
  k_one<F16, G, ZEROS, WN, WK><<<grid, 64 * WN * WK, WN * WK * STAGES * STAGE_BYTES + seg * 256, s>>>(
      x, ldx, codes, scales, zeros, y, ldy, n, k, group, seg);
  return hipGetLastError();
}

template <bool F16, int G, bool ZEROS>
hipError_t one(const void* x, long long ldx, const uint8_t* codes, const void* scales, const uint8_t* zeros, void* y,
               long long ldy, int m, int n, int k, int group, hipStream_t s) {
  const int tiles = (n + 15) / 16 * m;  // over all rows of x
  const int chunks = (k + CHUNK - 1) / CHUNK;
  // Enough tiles for every compute unit: one wave a tile, and 4 tiles share what is read of x
  // (32768 x 4096: 17 us, 20 with 4 waves a tile).  Fewer: 4 waves a tile (4096 x 4096: 5.6
  // and 9.9 us), or 8 where the columns are long (4096 x 16384: 12.2 us, 13.5 with 4).
  if (tiles >= 2048) return one_as<F16, G, ZEROS, 4, 1>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, s);
  if (tiles > 256 || chunks < 96) return one_as<F16, G, ZEROS, 1, 4>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, s);
  return one_as<F16, G, ZEROS, 1, 8>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, s);
}

// 2 to 64 rows of x, in MT tiles of 16.  8 waves a workgroup, RT tiles of 16 rows of W each, all
// on the same columns: a stage is 2 chunks.  Codes come as in k_one, two stages ahead, images of
// 16 rows x 128 bytes with unit u of row r at u ^ (r/2 & 7); x comes through registers, one stage
// ahead, into LDS [32 units][16 MT rows], row i of unit u at i ^ (u & 15), in the order that the
// codes unpack to, with the sums over each scale's columns, which every tile needs.  While the
// matrix instructions of a step run, the codes of the next are unpacked and the sums of the last
// group scaled.  A wave reads x out of LDS for RT tiles at once (8 rows of x are 4 KiB a
// chunk, a tile's codes 1 KiB), and the whole workgroup reads it out of memory once: 256 rows
// of W a workgroup for more than 16 rows of x keep that to as much as the codes.  The columns
// are split over blockIdx.y: each split writes its own fp32 sums (`part`), which k_join adds in
// order; a single split writes y.
template <int SPC, int MT>
constexpr int XBytes = 32 * 16 * MT * 16 + 2 * SPC * 16 * MT * 4;  // a stage of x, and its sums
template <int CTRL>
__device__ __forceinline__ float add_lanes(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 15, 15, true));
}

template <bool F16, int G, bool ZEROS, int MT, int RT>
__global__ __launch_bounds__(512) void k_batch(const void* x, long long ldx, const uint8_t* codes, const void* scales,
                                               const uint8_t* zeros, void* y, long long ldy, int m, int n, int k,
                                               int group, int per, float* part_out) {
  using Y = Type<F16>;
  using T = typename Y::T;
  using Sc = Scales<F16, G, ZEROS>;
  constexpr int STEPS = 4 / Sc::SPC, ROWS = 16 * MT, SLOT = RT * 2048, COPIES = 2 * RT, XB = XBytes<Sc::SPC, MT>, AHEAD = 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane >> 4, r = lane & 15;
  const int row0 = (blockIdx.x * 8 + wave) * 16 * RT, groups = k / group, per_group = group / CHUNK;
  const int chunks = (k + CHUNK - 1) / CHUNK, c0 = blockIdx.y * per, c1 = min(chunks, c0 + per);
  char* mine = smem + 2 * XB + wave * AHEAD * SLOT;
  const uint64_t at0 = reinterpret_cast<uint64_t>(codes) + (uint64_t)min(row0, n - 1) * (k / 2);
  const uint64_t base = (uint64_t)__builtin_amdgcn_readfirstlane((unsigned)(at0 >> 32)) << 32 |
                        (unsigned)__builtin_amdgcn_readfirstlane((unsigned)at0);
  const auto buffer = __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void*>(base), 0, __builtin_amdgcn_readfirstlane(max(0, min(16 * RT, n - row0)) * (k / 2)),
      0x00020000);
  // lane (j, r) loads the scales of row r of tile j / 2, chunk j % 2 of the stage
  const int safe = min(row0 + (RT > 1 ? j / 2 * 16 : 0) + r, n - 1);
  const T* s_row = static_cast<const T*>(scales) + (size_t)safe * groups;
  const uint8_t* z_row = ZEROS ? zeros + (size_t)safe * groups : nullptr;

  auto copy = [&](int c, int slot) {
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int rr = i * 8 + (lane >> 3), u = (lane & 7) ^ (rr >> 1 & 7), off = rr * (k / 2) + c * (CHUNK / 2) + u * 16;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          buffer, (__attribute__((address_space(3))) void*)(mine + slot * SLOT + i * 1024), 16, c < c1 ? off : 0x7ffffff0,
          0, 0, 0);
    }
  };
  auto fetch = [&](int c) { return Sc::load(s_row, z_row, min(c + j % 2, chunks - 1), groups, per_group, group, k); };
  u32x4 xr[MT];
  auto load_x = [&](int c) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int p = tid + i * 512, row = min(p >> 5, m - 1), ks = min(c * CHUNK + (p & 31) * 8, k - 8);
      xr[i] = *reinterpret_cast<const u32x4*>(static_cast<const T*>(x) + row * ldx + ks);
    }
  };
  // x in LDS: this thread's place for the first tile, and where its lane finds step s of a chunk
  const int to = ((tid & 31) * ROWS + ((tid >> 5) ^ (tid & 15))) * 16;
  int from[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) from[s] = ((s * 4 + j) * ROWS + (r ^ (s * 4 + j))) * 16;
  auto store_x = [&](int c, char* xb) {
    if (c * CHUNK + 2 * CHUNK > k && c * CHUNK + (tid & 31) * 8 >= k) {
#pragma unroll
      for (int i = 0; i < MT; ++i) xr[i] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const u32x4 v = pairs(xr[i]);
      *reinterpret_cast<u32x4*>(xb + to + i * 256) = v;
      // the sum of x over a scale's columns: units of 8 lie in neighbouring lanes.  Without zeros
      // every code has the same offset, and the matrix instructions start at -offset sum x
      float s = Y::sum2(v[0], Y::sum2(v[1], Y::sum2(v[2], Y::sum2(v[3], 0.f))));
      s = add_lanes<0xb1>(s);                              // 1 lane apart
      s = add_lanes<0x4e>(s);                              // 2
      if constexpr (Sc::SPC < 4) s = add_lanes<0x141>(s);  // the other 4 of 8
      if constexpr (Sc::SPC < 2) s = add_lanes<0x140>(s);  // the other 8 of 16
      if (tid % (16 / Sc::SPC) == 0)
        reinterpret_cast<float*>(xb + 32 * ROWS * 16)[(tid & 31) / (16 / Sc::SPC) * ROWS + (tid >> 5) + i * 16] =
            ZEROS ? s : s * -Sc::OFFSET;
    }
  };

  f32x4 total[RT][MT];
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int t = 0; t < MT; ++t) total[a][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int lane_at = r * 128 + (r >> 1 & 7) * 16 + j * 4;

  const int stages = (c1 - c0 + 1) / 2;
  auto chunk_of = [&](int i) { return i < stages ? c0 + 2 * i : 1 << 20; };  // past the last stage nothing is read
  Sc f[AHEAD];
  copy(chunk_of(0), 0);
  f[0] = fetch(chunk_of(0));
  load_x(min(chunk_of(0), chunks - 1));
  asm volatile("" ::: "memory");  // in this order
  copy(chunk_of(1), 1);
  f[1] = fetch(chunk_of(1));
  int buf = 0;
  for (int i = 0; i < stages; i += AHEAD) {
#pragma unroll
    for (int slot = 0; slot < AHEAD; ++slot) {
      if (i + slot >= stages) break;
      const int at = chunk_of(i + slot);
      // loads return in order: the codes of this stage are older than its x, and of what is in
      // flight only the next stage's codes and scales are younger
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COPIES + Sc::LOADS) : "memory");
      char* xb = smem + buf * XB;
      store_x(at, xb);
      load_x(min(chunk_of(i + slot + 1), chunks - 1));
      // all codes of the stage, and x one step ahead of the matrix instructions: left to itself
      // the compiler reads right before each use and waits every time
      const char* img = mine + slot * SLOT;
      unsigned w[2][4][RT];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int a = 0; a < RT; ++a)
            w[u][s][a] = *reinterpret_cast<const unsigned*>(img + a * 2048 + (lane_at ^ ((u * 4 + s) * 16)));
      const Sc now = f[slot];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // x is written, and the codes' slot has been read
      copy(chunk_of(i + slot + AHEAD), slot);
      f[slot] = fetch(chunk_of(i + slot + AHEAD));
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");  // the barrier alone does not hold the compiler's loads back
      u32x4 xa[2][MT], b[2][RT];
      auto read_x = [&](int u, int s, u32x4* to) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
          to[t] = *reinterpret_cast<const u32x4*>(xb + from[s] + u * 16 * ROWS * 16 + t * 256);
      };
      read_x(0, 0, xa[0]);
#pragma unroll
      for (int a = 0; a < RT; ++a) b[0][a] = unpack<F16>(w[0][0][a]);
      Sc v[2][RT];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int a = 0; a < RT; ++a) v[u][a] = now.of(((a * 2 + u) * 16 + r) * 4, min(at + u, chunks - 1), groups);
      const float* xsum = reinterpret_cast<const float*>(xb + 32 * ROWS * 16) + j * 4;
      f32x4 part[2][RT][MT], sum[2][MT];
      // the sums of group g (of a scale's columns) for x's tile t, into the result
      auto finish = [&](int g, int t) {
#pragma unroll
        for (int a = 0; a < RT; ++a) {
          const float sc = v[g / Sc::SPC][a].scale(g % Sc::SPC), off = v[g / Sc::SPC][a].offset(g % Sc::SPC);
          const f32x4 p = part[g & 1][a][t];
#pragma unroll
          for (int e = 0; e < 4; ++e) total[a][t][e] += sc * (ZEROS ? p[e] - off * sum[g & 1][t][e] : p[e]);
        }
      };
#pragma unroll
      for (int us = 0; us < 8; ++us) {  // a chunk past the row's end has zeros in x
        const int g = us / STEPS, step = us % STEPS;
        __builtin_amdgcn_sched_barrier(0);
        if (us < 7) read_x((us + 1) / 4, (us + 1) % 4, xa[(us + 1) & 1]);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if (step == 0) {
            sum[g & 1][t] = *reinterpret_cast<const f32x4*>(xsum + g * ROWS + t * 16);
#pragma unroll
            for (int a = 0; a < RT; ++a) part[g & 1][a][t] = ZEROS ? f32x4{0.f, 0.f, 0.f, 0.f} : sum[g & 1][t];
          }
#pragma unroll
          for (int a = 0; a < RT; ++a) part[g & 1][a][t] = Y::mfma(xa[us & 1][t], b[us & 1][a], part[g & 1][a][t]);
        }
        // meanwhile the vector unit unpacks the next step's codes and scales the last group's sums
        if (us < 7) {
#pragma unroll
          for (int a = 0; a < RT; ++a) b[(us + 1) & 1][a] = unpack<F16>(w[(us + 1) / 4][(us + 1) % 4][a]);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
          if (g && t * STEPS / MT == step) finish(g - 1, t);
        if constexpr (MT * RT >= 4) {
          __builtin_amdgcn_sched_group_barrier(0x100, MT, 0);  // reads of LDS
#pragma unroll
          for (int i = 0; i < MT * RT; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                          // a matrix instruction,
            __builtin_amdgcn_sched_group_barrier(0x002, (RT * 8 + MT * RT) / (MT * RT) + 1, 0);  // vector ones
          }
        }
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) finish(2 * Sc::SPC - 1, t);
      buf ^= 1;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the workgroup's LDS
#pragma unroll
  for (int a = 0; a < RT; ++a) {
    const int row = row0 + a * 16 + r;
    if (row >= n) continue;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int xrow = t * 16 + j * 4 + e;
        if (xrow >= m) continue;
        if (part_out) part_out[((size_t)blockIdx.y * m + xrow) * n + row] = total[a][t][e];
        else static_cast<T*>(y)[xrow * ldy + row] = (T)total[a][t][e];
      }
  }
}

// y = the sum of the splits, in order.
template <typename T>
__global__ __launch_bounds__(256) void k_join(const float* __restrict__ part, int splits, int m, int n,
                                              T* __restrict__ y, long long ldy) {
  const int row = blockIdx.x * 256 + threadIdx.x, xrow = blockIdx.y;
  if (row >= n) return;
  const float* from = part + (size_t)xrow * n + row;
  const size_t step = (size_t)m * n;
  float s = 0.f;
  for (int i = 0; i < splits; i += 8) {  // 8 loads in flight (8 x 1024 x 16384, 32 splits: 9.5 us for 16.9)
    float v[8];
#pragma unroll
    for (int o = 0; o < 8; ++o) v[o] = i + o < splits ? from[(i + o) * step] : 0.f;
#pragma unroll
    for (int o = 0; o < 8; ++o) s += v[o];
  }
  y[xrow * ldy + row] = (T)s;
}

template <bool F16, int G, bool ZEROS, int MT, int RT>
hipError_t batch_as(const void* x, long long ldx, const uint8_t* codes, const void* scales, const uint8_t* zeros,
                    void* y, long long ldy, int m, int n, int k, int group, int splits, float* part, hipStream_t s) {
  constexpr size_t lds = 2 * XBytes<Scales<F16, G, ZEROS>::SPC, MT> + 8 * 2 * RT * 2048;
  const int chunks = (k + CHUNK - 1) / CHUNK, per = ((chunks + splits - 1) / splits + 1) / 2 * 2;
  const dim3 grid((n + 128 * RT - 1) / (128 * RT), splits);
  k_batch<F16, G, ZEROS, MT, RT><<<grid, 512, lds, s>>>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, per,
                                                    splits > 1 ? part : nullptr);
  if (splits > 1) {
    using T = typename Type<F16>::T;
    k_join<T><<<dim3((n + 255) / 256, m), 256, 0, s>>>(part, splits, m, n, static_cast<T*>(y), ldy);
  }
  return hipGetLastError();
}

template <bool F16, int G, bool ZEROS>
hipError_t run(const void* x, long long ldx, const uint8_t* codes, const void* scales, const uint8_t* zeros, void* y,
               long long ldy, int m, int n, int k, int group, int splits, float* part, bool each, hipStream_t s) {
  if (each) return one<F16, G, ZEROS>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, s);
  if (m <= 16) return batch_as<F16, G, ZEROS, 1, 1>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, splits, part, s);
  if (m <= 32) return batch_as<F16, G, ZEROS, 2, 2>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, splits, part, s);
  return batch_as<F16, G, ZEROS, 4, 2>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, splits, part, s);
}

template <bool F16>
hipError_t launch(const void* x, long long ldx, const uint8_t* codes, const void* scales, const uint8_t* zeros,
                  void* y, long long ldy, int m, int n, int k, int group, int splits, float* part, bool each,
                  hipStream_t s) {
  const int g = group % CHUNK == 0 ? 1 : k < CHUNK ? 0 : group == 64 ? 2 : group == 32 ? 4 : 0;
#define RUN(G)                                                                                                \
  (zeros ? run<F16, G, true>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, splits, part, each, s)     \
         : run<F16, G, false>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, splits, part, each, s))
  return g == 1 ? RUN(1) : g == 2 ? RUN(2) : g == 4 ? RUN(4) : RUN(0);
#undef RUN
}

int refuse(const char* why) {
  snprintf(g_err, sizeof(g_err), "%s", why);
  return -1;
}

}  // namespace

// One call's tensors and sizes (ops/gemv.py packs the same fields in the same order).
struct tkv_args {
  int dev, f16, m, n, k, group;
  int splits;            // 0: each row of x by itself, k_one; else together, k_batch, the columns split
  long long ldx, ldy;    // row strides, elements
  const void *x, *codes, *scales;  // codes [n][k/2], the lower half of a byte first; scales [n][k/group] of x's type
  const void* zeros;     // [n][k/group] bytes, or null for 8
  void *y, *part;        // part: splits x m x n fp32 sums
  void* stream;
};

extern "C" int tkv_args_size() { return (int)sizeof(tkv_args); }

// y[m][n] = x[m][k] W^T, queued on a->stream; nothing waits for it.  0, or -1 / a HIP error with
// tkv_last_error() set.
extern "C" int tkv_gemv_w4(const tkv_args* a) {
  const int dev = a->dev, m = a->m, n = a->n, k = a->k, group = a->group, splits = a->splits;
  const long long ldx = a->ldx, ldy = a->ldy;
  const void *x = a->x, *codes = a->codes, *scales = a->scales, *zeros = a->zeros;
  void *y = a->y, *part = a->part;
  if (m < 1 || m > 64) return refuse("1 to 64 rows of x");
  if (n < 1 || n > (1 << 24)) return refuse("1 to 2^24 rows of weights");
  if (group < 32 || group % 32 || k < group || k % group || k > (1 << 20))
    return refuse("the group must be a multiple of 32 that divides k, and k at most 2^20");
  if (ldx < k || (ldx & 7) || (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(codes) & 15))
    return refuse("rows of x and of the codes must be 16-byte aligned");
  if (ldy < n) return refuse("y's row stride is below its width");
  if (splits < 0 || splits > 64 || (splits > 1 && !part)) return refuse("0 to 64 splits, with room for their sums");
  int prev = 0;
  hipError_t e = hipGetDevice(&prev);
  if (e == hipSuccess && prev != dev) e = hipSetDevice(dev);
  if (e == hipSuccess) {
    const auto s = static_cast<hipStream_t>(a->stream);
    const auto *c = static_cast<const uint8_t*>(codes), *z = static_cast<const uint8_t*>(zeros);
    float* p = static_cast<float*>(part);
    e = a->f16 ? launch<true>(x, ldx, c, scales, z, y, ldy, m, n, k, group, splits, p, splits == 0, s)
               : launch<false>(x, ldx, c, scales, z, y, ldy, m, n, k, group, splits, p, splits == 0, s);
    if (prev != dev) {
      const hipError_t back = hipSetDevice(prev);
      if (e == hipSuccess) e = back;
    }
  }
  if (e == hipSuccess) return 0;
  snprintf(g_err, sizeof(g_err), "gemv: %s (%d)", hipGetErrorString(e), (int)e);
  return (int)e;
}
