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
// C ABI for ctypes: triton_kubernetes_amd/ops/gemv.py.

#include <hip/hip_runtime.h>

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
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int up = Y::LOW - 4 * i;
    const unsigned s = up >= 0 ? w << (up & 31) : w >> (-up & 31);
    r[i] = (s & Y::MASK) | Y::SIXTEEN;
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

constexpr int WAVES = 8;
constexpr int CHUNK = 128;  // codes of a row that a wave reads at once: 16 bytes a lane, 64 a row

// 16 rows of W a workgroup, the chunks of K dealt out to its waves; MT tiles of 16 rows of x.
// Lane (j, r) = (lane / 16, lane % 16) reads codes of row r, and holds sums of that row with
// rows 4j..4j+3 of each tile of x.
template <bool F16, int MT>
__global__ __launch_bounds__(64 * WAVES) void k_gemv(const void* __restrict__ x, long long ldx,
                                                     const uint8_t* __restrict__ codes,
                                                     const void* __restrict__ scales,
                                                     const uint8_t* __restrict__ zeros, void* __restrict__ y,
                                                     long long ldy, int m, int n, int k, int group) {
  using Y = Type<F16>;
  using T = typename Y::T;
  __shared__ float sum[WAVES][MT * 4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane >> 4, r = lane & 15;
  const int row = blockIdx.x * 16 + r, groups = k / group;
  const int safe = min(row, n - 1);
  const uint8_t* c_row = codes + (size_t)safe * (k / 2);
  const T* s_row = static_cast<const T*>(scales) + (size_t)safe * groups;
  const uint8_t* z_row = zeros ? zeros + (size_t)safe * groups : nullptr;

  f32x4 total[MT], part[MT], sx[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) total[t] = part[t] = sx[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const u32x4 ones = {Y::ONES, Y::ONES, Y::ONES, Y::ONES};
  const u32x4 none = {0, 0, 0, 0};
  const int chunks = (k + CHUNK - 1) / CHUNK;
  for (int c = wave; c < chunks; c += WAVES) {
    const int k0 = c * CHUNK;
    u32x4 w = none;
    if (k0 + j * 32 < k) w = *reinterpret_cast<const u32x4*>(c_row + (k0 + j * 32) / 2);
    w = exchange(w);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int ks = k0 + s * 32;
      if (ks >= k) break;
      const u32x4 b = unpack<F16>(w[s]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        u32x4 a = none;
        if (t * 16 + r < m)
          a = pairs(*reinterpret_cast<const u32x4*>(static_cast<const T*>(x) + (t * 16 + r) * ldx + ks + j * 8));
        part[t] = Y::mfma(a, b, part[t]);
        sx[t] = Y::mfma(a, ones, sx[t]);
      }
      if ((ks + 32) % group == 0 || s == 3 || ks + 32 >= k) {  // the group ends, or the wave's part of it
        const int g = ks / group;
        const float sc = (float)s_row[g], off = 16.f + (z_row ? (float)z_row[g] : 8.f);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          total[t] += sc * (part[t] - off * sx[t]);
          part[t] = sx[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[wave][t * 4 + e][lane] = total[t][e];
  __syncthreads();
  for (int i = wave; i < MT * 4; i += WAVES) {
    float s = 0.f;
#pragma unroll
    for (int o = 0; o < WAVES; ++o) s += sum[o][i][lane];
    const int xr = (i >> 2) * 16 + j * 4 + (i & 3);
    if (xr < m && row < n) static_cast<T*>(y)[xr * ldy + row] = (T)s;
  }
}

template <bool F16>
hipError_t launch(const void* x, long long ldx, const uint8_t* codes, const void* scales, const uint8_t* zeros,
                  void* y, long long ldy, int m, int n, int k, int group, hipStream_t s) {
  const unsigned grid = (n + 15) / 16;
  if (m <= 16) k_gemv<F16, 1><<<grid, 64 * WAVES, 0, s>>>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group);
  else if (m <= 32) k_gemv<F16, 2><<<grid, 64 * WAVES, 0, s>>>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group);
  else k_gemv<F16, 4><<<grid, 64 * WAVES, 0, s>>>(x, ldx, codes, scales, zeros, y, ldy, m, n, k, group);
  return hipGetLastError();
}

int refuse(const char* why) {
  snprintf(g_err, sizeof(g_err), "%s", why);
  return -1;
}

}  // namespace

// y[m][n] = x[m][k] W^T, queued on `stream` of device `dev`; nothing waits for it.  codes
// [n][k/2] (the lower half of a byte first), scales [n][k/group] of x's type, zeros
// [n][k/group] bytes or null for 8.  0, or -1 / a HIP error with tkv_last_error() set.
extern "C" int tkv_gemv_w4(int dev, int f16, const void* x, long long ldx, const void* codes, const void* scales,
                           const void* zeros, void* y, long long ldy, int m, int n, int k, int group, void* stream) {
  if (m < 1 || m > 64) return refuse("1 to 64 rows of x");
  if (n < 1 || n > (1 << 24)) return refuse("1 to 2^24 rows of weights");
  if (group < 32 || group % 32 || k < group || k % group || k > (1 << 20))
    return refuse("the group must be a multiple of 32 that divides k, and k at most 2^20");
  if (ldx < k || (ldx & 7) || (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(codes) & 15))
    return refuse("rows of x and of the codes must be 16-byte aligned");
  if (ldy < n) return refuse("y's row stride is below its width");
  int prev = 0;
  hipError_t e = hipGetDevice(&prev);
  if (e == hipSuccess && prev != dev) e = hipSetDevice(dev);
  if (e == hipSuccess) {
    const auto s = static_cast<hipStream_t>(stream);
    const auto *c = static_cast<const uint8_t*>(codes), *z = static_cast<const uint8_t*>(zeros);
    e = f16 ? launch<true>(x, ldx, c, scales, z, y, ldy, m, n, k, group, s)
            : launch<false>(x, ldx, c, scales, z, y, ldy, m, n, k, group, s);
    if (prev != dev) {
      const hipError_t back = hipSetDevice(prev);
      if (e == hipSuccess) e = back;
    }
  }
  if (e == hipSuccess) return 0;
  snprintf(g_err, sizeof(g_err), "gemv: %s (%d)", hipGetErrorString(e), (int)e);
  return (int)e;
}
