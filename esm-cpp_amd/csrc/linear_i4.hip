// Linears with 4-bit weights for gfx950: y = x W^T + bias, W[n, k] = code[n, k]
// * scale[n, k / group], codes in -8 .. 7, activations and outputs fp32, fp16 or
// bf16, sums in fp32.
//
// A code is an fp16 number as it stands, so the products run on fp16 MFMA with
// the weight operand exact: for fp16 activations directly, for bf16 ones (8
// significant bits) after a power of two that brings the largest of a row (of 128
// of its inputs, in the kernel for few rows) to [2^14, 2^15), and for fp32 ones as
// hi + lo fp16 parts (22 significant bits) of the same scaled value, two MFMAs per
// product. What lies far below the largest is off by half of fp16's smallest step
// at most, 2^-39 of the largest. A group's sum leaves the matrix cores before it is multiplied by its scale (and by the
// power of two's inverse): one fused multiply-add per output, group and row.
//
// Weights lie in tiles of 16 outputs x 128 inputs, 1 KB, in the order of the
// operand registers of v_mfma_f32_16x16x32_f16: lane n % 16 + 16 kq holds 16
// bytes, whose dword j has inputs 32 j + 8 kq .. + 8. Input 2 p of the eight is
// nibble p and input 2 p + 1 nibble p + 4, so that one and-or turns two codes
// into the fp16 pair 1024 + u (or 1024 + 16 u), and one packed add (fma) into
// the codes: nine instructions for eight weights.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "kernels.hpp"

namespace esm_gfx950 {

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kTileN = 16, kTileK = 128;

// Elements from one plane of split activations to the next: rows in sixteens.
__host__ __device__ inline size_t plane_elems(int M, int ldp) { return (static_cast<size_t>(M) + 15) / 16 * 16 * ldp; }

// Eight codes of one dword as fp16.
__device__ __forceinline__ f16x8 unpack_codes(uint32_t w) {
  const f16x2 k1032 = {static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
  const f16x2 k16th = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
  const f16x2 k72 = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
  const uint32_t v = w >> 8;
  const f16x2 a = __builtin_bit_cast(f16x2, (w & 0x000f000fu) | 0x64006400u) + k1032;
  const f16x2 b = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & 0x00f000f0u) | 0x64006400u), k16th, k72);
  const f16x2 c = __builtin_bit_cast(f16x2, (v & 0x000f000fu) | 0x64006400u) + k1032;
  const f16x2 d = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (v & 0x00f000f0u) | 0x64006400u), k16th, k72);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Element types of the activations and outputs.
template <int DT>
struct Elem;
template <>
struct Elem<kTypeF32> {
  using T = float;
  static constexpr int kPlanes = 2;
};
template <>
struct Elem<kTypeF16> {
  using T = _Float16;
  static constexpr int kPlanes = 1;
};
template <>
struct Elem<kTypeBF16> {
  using T = __bf16;
  static constexpr int kPlanes = 1;
};

// Eight consecutive inputs of a row from k on, zeros past K (and for row null).
template <class T>
__device__ __forceinline__ void load8(const T* row, int k, int K, bool vec, T (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = static_cast<T>(0.0f);
  if (!row) return;
  if (vec && k + 8 <= K) {
    constexpr int kPieces = sizeof(T) * 8 / 16;
    uint4 p[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) p[i] = reinterpret_cast<const uint4*>(row + k)[i];
    __builtin_memcpy(x, p, sizeof(p));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) x[i] = row[k + i];
  }
}

// Four consecutive outputs of row m from column n on, with their bias.
template <class T>
__device__ __forceinline__ void store4(const LinearI4Args& p, int m, int n, f32x4 sum) {
  if (m >= p.M) return;
  T* c = static_cast<T*>(p.C) + static_cast<size_t>(m) * p.ldc + n;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < p.N) c[i] = static_cast<T>(sum[i] + (p.bias ? p.bias[n + i] : 0.0f));
}

// The exponent e for which amax * 2^e lies in [2^14, 2^15) (amax finite;
// limited to what 2^e and 2^-e can be).
__device__ __forceinline__ int row_exponent(float amax) {
  return amax > 0.0f ? max(-120, min(120, 15 - __builtin_amdgcn_frexp_expf(amax))) : 0;
}

// Eight values of a row's 128, the others in the lane's group of 16, as fp16 hi
// (and lo) operands of the scaled values; *inv receives the scale's inverse. An
// infinity stays one (its lo part is zero), the others are scaled without it.
template <int PL>
__device__ __forceinline__ void split_scaled(const float (&x)[8], uint4 (&out)[PL], float* inv) {
  auto over_lanes = [](float v) {
    v = fmaxf(v, lane_dpp<0x128>(v));  // row_ror:8
    v = fmaxf(v, lane_dpp<0x124>(v));  // row_ror:4
    v = fmaxf(v, lane_dpp<0x4e>(v));   // quad_perm [2, 3, 0, 1]
    return fmaxf(v, lane_dpp<0xb1>(v));  // quad_perm [1, 0, 3, 2]
  };
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i += 2)  // one instruction for two (fmaxf quiets its operands first)
    asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(amax) : "v"(x[i]), "v"(x[i + 1]));
  amax = over_lanes(amax);
  const bool finite = amax < INFINITY;
  if (__builtin_amdgcn_ballot_w64(!finite)) {
    float fmax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) fmax = fmaxf(fmax, fabsf(x[i]) < INFINITY ? fabsf(x[i]) : 0.0f);
    amax = over_lanes(fmax);
  }
  const int e = row_exponent(amax);
  const float mul = __builtin_amdgcn_ldexpf(1.0f, e);
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) split_pair(x[2 * i] * mul, x[2 * i + 1] * mul, &h[i], &l[i]);
  out[0] = make_uint4(h[0], h[1], h[2], h[3]);
  if constexpr (PL == 2) {
    if (__builtin_amdgcn_ballot_w64(!finite)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (fabsf(x[i]) == INFINITY) l[i >> 1] &= i & 1 ? 0x0000ffffu : 0xffff0000u;
    }
    out[PL - 1] = make_uint4(l[0], l[1], l[2], l[3]);
  }
  *inv = __builtin_amdgcn_ldexpf(1.0f, -e);
}

}  // namespace

// ------------------------------------------------------------- up to 16 rows
// One workgroup: all rows x 16 NT outputs, its waves taking the 128-input tiles in
// turn and adding up through LDS. The workgroup splits the activations into LDS
// once, every lane eight inputs of its own (as operands loaded and split in each
// lane, 16 lanes would do one row's work over again: 1 x 10,240 x 2,560 13 us
// instead of 8), while the first tile's codes and scales are on their way; a
// tile's are loaded while the tile before is computed. D = W x^T, so that a
// lane's outputs are four consecutive ones of one row. 1 x 1,280 x 1,280 takes 4 us,
// a launch and two trips to memory; 14 MB of 10,240 x 2,560 9, at 1.6 TB/s, a wave's
// two tiles one after the other.
template <int DT, int NT, int GJ>  // GJ: 32-input steps of a group within a tile (1, 2 or 4)
__global__ __launch_bounds__(1024) void linear_i4_rows_kernel(LinearI4Args p, int chunk) {
  using T = typename Elem<DT>::T;
  constexpr int PL = Elem<DT>::kPlanes;
  constexpr int kTileBytes = PL * 256;  // a row's 128 inputs
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int lr = lane & 15, kq = lane >> 4;
  const int tn0 = blockIdx.x * NT, tiles_n = (p.N + kTileN - 1) / kTileN;
  const int pitch = chunk * kTileBytes + 16;  // rows of 16-byte pieces on distinct banks
  float* inv = reinterpret_cast<float*>(lds + p.M * pitch);  // [chunk][M]
  struct Tile {
    u32x4 w[NT];
    f32x4 s[NT][4 / GJ];
  };
  auto load = [&](int kt, Tile& t) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int tn = min(tn0 + nt, tiles_n - 1);
      t.w[nt] = reinterpret_cast<const u32x4*>(p.W)[(static_cast<size_t>(tn) * p.tiles_k + kt) * 64 + lane];
#pragma unroll
      for (int g = 0; g < 4 / GJ; ++g) {
        const int group = min((kt * kTileK + g * 32 * GJ) / p.group, p.groups - 1);
        t.s[nt][g] = *reinterpret_cast<const f32x4*>(p.scales + (static_cast<size_t>(tn) * p.groups + group) * kTileN + 4 * kq);
      }
    }
  };
  f32x4 total[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) total[nt] = f32x4{0.f, 0.f, 0.f, 0.f};

  Tile next;
  if (wave < p.tiles_k) load(wave, next);
  for (int c0 = 0; c0 < p.tiles_k; c0 += chunk) {  // chunk: a multiple of the waves, or all tiles
    const int n = min(chunk, p.tiles_k - c0);
    if (c0 > 0) __syncthreads();
    // 16 lanes to a tile of a row.
    for (int u = wave * 4 + kq; u < n * p.M; u += waves * 4) {
      const int tile = u / p.M, m = u - tile * p.M;
      T x[8];
      load8<T>(static_cast<const T*>(p.A) + static_cast<size_t>(m) * p.lda, (c0 + tile) * kTileK + 8 * lr, p.K, p.vec_a, x);
      uint4 out[PL];
      float unit = 1.0f;
      if constexpr (DT == kTypeF16) {
        __builtin_memcpy(&out[0], x, 16);
      } else {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(x[i]);
        split_scaled<PL>(f, out, &unit);
      }
      uint8_t* at = lds + m * pitch + tile * kTileBytes + lr * 16;
#pragma unroll
      for (int pl = 0; pl < PL; ++pl) *reinterpret_cast<uint4*>(at + pl * 256) = out[pl];
      if (lr == 0) inv[tile * p.M + m] = unit;
    }
    __syncthreads();
    const int m = min(lr, p.M - 1);  // lanes past the last row take it again; their outputs are not stored
    for (int tile = wave; tile < n; tile += waves) {
      const Tile t = next;
      if (c0 + tile + waves < p.tiles_k) load(c0 + tile + waves, next);
      const uint8_t* at = lds + m * pitch + tile * kTileBytes + kq * 16;
      f16x8 a[4][PL];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int pl = 0; pl < PL; ++pl) a[j][pl] = *reinterpret_cast<const f16x8*>(at + pl * 256 + j * 64);
      const float unit = inv[tile * p.M + m];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        f32x4 acc;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f16x8 wf = unpack_codes(t.w[nt][j]);
          acc = mma(wf, a[j][0], j % GJ == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc);
          if constexpr (PL == 2) acc = mma(wf, a[j][PL - 1], acc);
          if ((j + 1) % GJ == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) total[nt][i] = __builtin_fmaf(acc[i], t.s[nt][j / GJ][i] * unit, total[nt][i]);
          }
        }
      }
    }
  }

  // The waves' sums meet in LDS and are added in the waves' order.
  __syncthreads();
  f32x4* out4 = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) out4[(wave * NT + nt) * 64 + lane] = total[nt];
  __syncthreads();
  for (int u = wave; u < NT; u += waves) {
    f32x4 sum = out4[u * 64 + lane];
    for (int w = 1; w < waves; ++w) sum += out4[(w * NT + u) * 64 + lane];
    store4<T>(p, lr, (tn0 + u) * kTileN + 4 * kq, sum);
  }
}

// ------------------------------------------------------------- many rows
// Activations as the matrix cores take them, written once for every column tile:
// fp16 planes (hi, and lo for fp32) of M rows, rounded up to 16, of ldp inputs,
// zeros past K, a row scaled by the power of two that brings its largest to
// [2^14, 2^15), the power's inverse in inv; fp16 rows as they are, where their
// alignment or length keeps the kernels from reading them in place. One workgroup
// per row. Row after row for the GEMM; for the small tiles (TILED) 16 rows x 32
// inputs after each other in the lanes' order, which the kernel loads in whole
// kilobytes (row by row, four neighbouring lanes' 16 bytes lie in four rows and
// take four accesses). The 16 rows of a tile are then one XCD's, whose L2 joins
// their pieces.
template <int DT, bool TILED>
__global__ __launch_bounds__(256) void linear_i4_split_kernel(LinearI4Args p, uint16_t* planes, float* inv, int ldp) {
  using T = typename Elem<DT>::T;
  __shared__ float part[4];
  const int m = TILED ? (blockIdx.x % 8 + blockIdx.x / 128 * 8) * 16 + blockIdx.x / 8 % 16 : blockIdx.x;
  if (m >= p.M) return;
  const T* row = static_cast<const T*>(p.A) + static_cast<size_t>(m) * p.lda;
  uint16_t* hi = planes + (TILED ? static_cast<size_t>(m / 16) * 16 * ldp + m % 16 * 8 : static_cast<size_t>(m) * ldp);
  uint16_t* lo = hi + plane_elems(p.M, ldp);
  float mul = 1.0f;
  if constexpr (DT != kTypeF16) {
    float amax = 0.0f;
    for (int k = threadIdx.x * 8; k < p.K; k += 2048) {
      T x[8];
      load8<T>(row, k, p.K, p.vec_a, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = fabsf(static_cast<float>(x[i]));
        amax = fmaxf(amax, v < INFINITY ? v : 0.0f);
      }
    }
    amax = wave_max(amax);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
    __syncthreads();
    const int e = row_exponent(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
    mul = __builtin_amdgcn_ldexpf(1.0f, e);
    if (threadIdx.x == 0) inv[m] = __builtin_amdgcn_ldexpf(1.0f, -e);
  }
  for (int k = threadIdx.x * 8; k < ldp; k += 2048) {
    T x[8];
    load8<T>(row, k, p.K, p.vec_a, x);
    f16x8 h, l;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = static_cast<float>(x[i]) * mul;
      h[i] = static_cast<_Float16>(v);
      l[i] = static_cast<_Float16>(fabsf(v) < INFINITY ? v - static_cast<float>(h[i]) : 0.0f);
    }
    const size_t at = TILED ? static_cast<size_t>(k) * 16 : k;  // eight inputs of 16 rows: 128 elements
    *reinterpret_cast<f16x8*>(hi + at) = h;
    if constexpr (Elem<DT>::kPlanes == 2) *reinterpret_cast<f16x8*>(lo + at) = l;
  }
}

// 16 MT rows x 16 NT outputs per workgroup, for grids that larger tiles would
// leave empty: the waves take the 128-input tiles in turn, straight from memory
// into their operand registers, and add up through LDS. 16 x 32 tiles wait for
// each tile's loads and leave the CU to two or three other workgroups meanwhile
// (67 fp32 rows of 3,840 x 1,280 11.1 us a call, 14.5 with the next tile's loads in
// flight and one workgroup a CU); 32 x 64 ones (one plane only) have those in flight.
// in_place: planes are the caller's fp16 rows, not the split kernel's. A load then
// takes 256 bytes of four rows, and a wave turns its tile round through its own
// part of LDS (301 rows of 1,280 x 5,120 14.1 us; loaded in the operands' places,
// four neighbouring lanes in four rows, 16.5).
template <int DT, int MT, int NT, int GJ>
__global__ __launch_bounds__(512, NT == 2 ? 4 : 2) void linear_i4_mid_kernel(
    LinearI4Args p, const uint16_t* planes, const float* inv, int ldp, bool in_place) {
  using T = typename Elem<DT>::T;
  constexpr int PL = Elem<DT>::kPlanes;
  extern __shared__ float red[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int lr = lane & 15, kq = lane >> 4;
  const int cols = (p.N + 16 * NT - 1) / (16 * NT), tiles_n = (p.N + kTileN - 1) / kTileN;
  const int tn0 = blockIdx.x % cols * NT, m0 = blockIdx.x / cols * (16 * MT);
  constexpr bool kAhead = NT > 2;
  const bool rowwise = DT == kTypeF16 && in_place;
  const uint16_t* rows[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
    rows[mt] = planes + (rowwise ? static_cast<size_t>(m0 + 16 * mt) * ldp + 8 * lr
                                 : static_cast<size_t>(min(m0 / 16 + mt, (p.M - 1) / 16)) * 16 * ldp + 8 * lane);
  const size_t plane = plane_elems(p.M, ldp);
  struct Tile {
    u32x4 w[NT];
    f32x4 s[NT][4 / GJ];
    f16x8 a[MT][4][PL];
  };
  auto load = [&](int kt, Tile& t) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int tn = min(tn0 + nt, tiles_n - 1);
      t.w[nt] = reinterpret_cast<const u32x4*>(p.W)[(static_cast<size_t>(tn) * p.tiles_k + kt) * 64 + lane];
#pragma unroll
      for (int g = 0; g < 4 / GJ; ++g) {
        const int group = min((kt * kTileK + g * 32 * GJ) / p.group, p.groups - 1);
        t.s[nt][g] = *reinterpret_cast<const f32x4*>(p.scales + (static_cast<size_t>(tn) * p.groups + group) * kTileN + 4 * kq);
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int pl = 0; pl < PL; ++pl)
          t.a[mt][j][pl] = *reinterpret_cast<const f16x8*>(
              rowwise ? rows[mt] + min(4 * j + kq, p.M - 1 - m0 - 16 * mt) * static_cast<ptrdiff_t>(ldp) + kt * kTileK
                      : rows[mt] + pl * plane + (static_cast<size_t>(kt) * 4 + j) * 512);
  };
  f32x4 total[NT][MT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) total[nt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  Tile next;
  if (kAhead && wave < p.tiles_k) load(wave, next);
  for (int kt = wave; kt < p.tiles_k; kt += waves) {
    if (!kAhead) load(kt, next);
    Tile t = next;
    if (rowwise) {  // row 4 j + kq, inputs 8 lr .. + 8 to row lr, inputs 32 j + 8 kq .. + 8
      uint8_t* own = reinterpret_cast<uint8_t*>(red) + wave * (MT * 4096);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f16x8*>(own + mt * 4096 + (4 * j + kq) * 256 + (lr ^ (4 * j + kq)) * 16) = t.a[mt][j][0];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          t.a[mt][j][0] = *reinterpret_cast<const f16x8*>(own + mt * 4096 + lr * 256 + ((4 * j + kq) ^ lr) * 16);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if (kAhead && kt + waves < p.tiles_k) load(kt + waves, next);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      f32x4 acc[MT];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f16x8 wf = unpack_codes(t.w[nt][j]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          acc[mt] = mma(wf, t.a[mt][j][0], j % GJ == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[mt]);
          if constexpr (PL == 2) acc[mt] = mma(wf, t.a[mt][j][PL - 1], acc[mt]);
        }
        if ((j + 1) % GJ == 0) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              total[nt][mt][i] = __builtin_fmaf(acc[mt][i], t.s[nt][j / GJ][i], total[nt][mt][i]);
        }
      }
    }
  }
  if (rowwise) __syncthreads();  // the waves' rows lie where the sums go
  f32x4* out4 = reinterpret_cast<f32x4*>(red);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) out4[(wave * NT * MT + nt * MT + mt) * 64 + lane] = total[nt][mt];
  __syncthreads();
  for (int u = wave; u < NT * MT; u += waves) {
    f32x4 sum = out4[u * 64 + lane];
    for (int w = 1; w < waves; ++w) sum += out4[(w * NT * MT + u) * 64 + lane];
    const int m = m0 + 16 * (u % MT) + lr;
    const float unit = inv ? inv[min(m, p.M - 1)] : 1.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] *= unit;
    store4<T>(p, m, (tn0 + u / MT) * kTileN + 4 * kq, sum);
  }
}

// 64 x 256 outputs per workgroup, 64 x 64 per wave on v_mfma_f32_32x32x16_f16:
// activations through LDS by direct loads, 64 inputs a stage, two stages; codes
// straight from global memory into the operand registers, the next 128 inputs'
// on their way. D has outputs across lanes: a group's scale is one register per
// 32 columns. The tile is wide because a row of split fp32 activations costs four
// bytes an input and a column of codes half a byte, and low so that two
// workgroups share a CU, one storing while the other multiplies: 4,099 x 5,120 x
// 1,280 took 139 us in 128 x 128 tiles, 132 in 128 x 256 and 129 in these. At
// 107 GFLOP of fp16 products (two per fp32 one) that is 830 TFLOP/s, 1,150 without
// the stores (84 MB, 12 us on their own) and the last, partly empty round.
constexpr int kGemmM = 64, kGemmN = 256, kGemmK = 64;
template <int DT, int GJ>  // GJ: 32-input steps of a group within 128 inputs
__global__ __launch_bounds__(256) void linear_i4_gemm_kernel(LinearI4Args p, const uint16_t* planes, const float* inv,
                                                             int ldp) {
  using T = typename Elem<DT>::T;
  constexpr int PL = Elem<DT>::kPlanes;
  constexpr int kPlaneBytes = kGemmM * kGemmK * 2;
  typedef float f32x16 __attribute__((ext_vector_type(16)));
  __shared__ __align__(1024) uint8_t stage[2][PL * kPlaneBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 31, half = lane >> 5;
  int m0, n0;
  tile_origin_of(blockIdx.x, p.M, p.N, kGemmM, kGemmN, &m0, &n0);

  // Direct loads: one instruction brings 8 rows of 64 inputs (1 KB); wave w loads
  // rows 16 w .. + 16. The 16-byte piece c of row r lies at c ^ (r / 2 % 8), so that
  // 16 rows' pieces fall on distinct banks.
  const uint32_t lds0 = lds_byte_addr(&stage[0][0]);
  uint32_t off[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = wave * 16 + i * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
    off[i] = static_cast<uint32_t>(min(r, p.M - 1 - m0)) * static_cast<uint32_t>(ldp * 2) + c * 16;
  }
  const size_t plane = PL == 2 ? plane_elems(p.M, ldp) : 0;
  auto load_stage = [&](int k0, int buf) {
#pragma unroll
    for (int pl = 0; pl < PL; ++pl) {
      const uint16_t* base = planes + pl * plane + static_cast<size_t>(m0) * ldp + k0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        lds_dma16(base, off[i], lds0 + buf * (PL * kPlaneBytes) + pl * kPlaneBytes + (wave * 16 + i * 8) * 128);
    }
  };

  // Codes: for 16 inputs s of 128, lane (n, half) takes dword s / 2 of storage lane
  // n % 16 + 16 (2 (s % 2) + half).
  const int tiles_n = (p.N + kTileN - 1) / kTileN;
  const u32x4* wp[2];
  const float* sp[2];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    const int tn = min((n0 + wave * 64 + nt * 32) / kTileN + (ln >> 4), tiles_n - 1);
    wp[nt] = reinterpret_cast<const u32x4*>(p.W) + static_cast<size_t>(tn) * p.tiles_k * 64 + (ln & 15) + 16 * half;
    sp[nt] = p.scales + static_cast<size_t>(tn) * p.groups * kTileN + (ln & 15);
  }
  u32x4 w[2][2], wnext[2][2];
  float s[2][4 / GJ], snext[2][4 / GJ];
  auto load_codes = [&](int kt, u32x4 (&to)[2][2], float (&st)[2][4 / GJ]) {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      to[nt][0] = wp[nt][static_cast<size_t>(kt) * 64];
      to[nt][1] = wp[nt][static_cast<size_t>(kt) * 64 + 32];
#pragma unroll
      for (int g = 0; g < 4 / GJ; ++g)
        st[nt][g] = sp[nt][static_cast<size_t>(min((kt * kTileK + g * 32 * GJ) / p.group, p.groups - 1)) * kTileN];
    }
  };

  f32x16 total[2][2], acc[2][2];
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int i = 0; i < 16; ++i) total[mt][nt][i] = acc[mt][nt][i] = 0.0f;

  load_stage(0, 0);
  load_codes(0, wnext, snext);
  for (int kt = 0; kt < p.tiles_k; ++kt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 64 inputs each
      // This stage has landed for every wave, and every wave is done with the other.
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (h == 0) {
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          w[nt][0] = wnext[nt][0];
          w[nt][1] = wnext[nt][1];
#pragma unroll
          for (int g = 0; g < 4 / GJ; ++g) s[nt][g] = snext[nt][g];
        }
        load_stage(kt * kTileK + kGemmK, 1);
      } else if (kt + 1 < p.tiles_k) {
        load_stage((kt + 1) * kTileK, 0);
        load_codes(kt + 1, wnext, snext);
      }
      // Each 16 inputs' operands are read and unpacked while the 16 before are on
      // the matrix cores.
      f16x8 a[2][2][PL], wf[2][2];
      auto operands = [&](int st) {
        const int step = h * 4 + st;  // of the 128 inputs' eight
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const int r = mt * 32 + ln;
          const uint8_t* at = stage[h] + r * 128 + (((2 * st + half) ^ ((r >> 1) & 7)) << 4);
#pragma unroll
          for (int pl = 0; pl < PL; ++pl) a[st & 1][mt][pl] = *reinterpret_cast<const f16x8*>(at + pl * kPlaneBytes);
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) wf[st & 1][nt] = unpack_codes(w[nt][step & 1][step >> 1]);
      };
      operands(0);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const int step = h * 4 + st;
        if (st < 3) operands(st + 1);
#pragma unroll
        for (int pl = 0; pl < PL; ++pl)
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
              acc[mt][nt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                  a[st & 1][mt][pl], wf[st & 1][nt], step % (2 * GJ) == 0 && pl == 0 ? f32x16{} : acc[mt][nt], 0, 0, 0);
        if (step % (2 * GJ) == 2 * GJ - 1) {
          const int g = step / (2 * GJ);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                total[mt][nt][i] = __builtin_fmaf(acc[mt][nt][i], s[nt][g], total[mt][nt][i]);
        }
#pragma unroll
        for (int i = 0; i < 4 * PL; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // an MFMA
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // an LDS read
          __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // vector instructions
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // A row's power of two once per row, and no conditions in whole tiles.
  const bool whole = m0 + kGemmM <= p.M && n0 + kGemmN <= p.N;
  const int n = n0 + wave * 64 + ln;
  float bias[2];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) bias[nt] = p.bias && n + nt * 32 < p.N ? p.bias[n + nt * 32] : 0.0f;
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int m = m0 + mt * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
      const float unit = inv ? inv[min(m, p.M - 1)] : 1.0f;
      T* c = static_cast<T*>(p.C) + static_cast<size_t>(m) * p.ldc + n;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const T y = static_cast<T>(__builtin_fmaf(total[mt][nt][i], unit, bias[nt]));
        if (whole || (m < p.M && n + nt * 32 < p.N)) c[nt * 32] = y;
      }
    }
}

namespace {

// The kernel of a group's 32-input steps within 128 inputs.
#define ESM_I4_BY_GROUP(KERNEL, ...)           \
  do {                                         \
    if (p.group == 32)                         \
      KERNEL(1, __VA_ARGS__);                  \
    else if (p.group == 64)                    \
      KERNEL(2, __VA_ARGS__);                  \
    else                                       \
      KERNEL(4, __VA_ARGS__);                  \
  } while (0)

template <int DT, int NT>
hipError_t launch_rows(const LinearI4Args& p, const LinearI4Plan& plan, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>((p.N + 16 * NT - 1) / (16 * NT)), block = 64 * plan.waves;
  const size_t row_bytes = static_cast<size_t>(plan.chunk) * (Elem<DT>::kPlanes * 256 + 4) + 16;
  const size_t lds = std::max(p.M * row_bytes, static_cast<size_t>(plan.waves) * NT * 1024);
  if (p.group == 64) {
    linear_i4_rows_kernel<DT, NT, 2><<<grid, block, lds, s>>>(p, plan.chunk);
  } else if (p.group != 32) {
    linear_i4_rows_kernel<DT, NT, 4><<<grid, block, lds, s>>>(p, plan.chunk);
  } else {
    if constexpr (NT == 1) linear_i4_rows_kernel<DT, 1, 1><<<grid, block, lds, s>>>(p, plan.chunk);
  }
  return hipGetLastError();
}

template <int DT, int MT, int NT, int GJ>
void launch_mid(const LinearI4Args& p, const LinearI4Plan& plan, const uint16_t* planes, const float* inv, int ldp,
                hipStream_t s) {
  const unsigned grid =
      static_cast<unsigned>((p.N + 16 * NT - 1) / (16 * NT)) * ((p.M + 16 * MT - 1) / (16 * MT));
  const size_t lds = static_cast<size_t>(plan.waves) * MT * std::max(NT * 1024, DT == kTypeF16 ? 4096 : 0);
  linear_i4_mid_kernel<DT, MT, NT, GJ><<<grid, 64 * plan.waves, lds, s>>>(p, planes, inv, ldp, plan.scratch_bytes == 0);
}

template <int DT>
hipError_t launch_typed(const LinearI4Args& p, const LinearI4Plan& plan, void* scratch, hipStream_t s) {
  if (plan.form == LinearI4Plan::kRows) return plan.col_tiles == 1 ? launch_rows<DT, 1>(p, plan, s) : launch_rows<DT, 2>(p, plan, s);
  int ldp = p.lda;
  const uint16_t* planes = static_cast<const uint16_t*>(p.A);
  const float* inv = nullptr;
  if (plan.scratch_bytes) {
    ldp = p.tiles_k * kTileK;
    auto* to = static_cast<uint16_t*>(scratch);
    auto* units = reinterpret_cast<float*>(to + Elem<DT>::kPlanes * plane_elems(p.M, ldp));
    if (plan.form == LinearI4Plan::kMid)
      linear_i4_split_kernel<DT, true><<<(p.M + 127) / 128 * 128, 256, 0, s>>>(p, to, units, ldp);
    else
      linear_i4_split_kernel<DT, false><<<p.M, 256, 0, s>>>(p, to, units, ldp);
    planes = to;
    inv = DT == kTypeF16 ? nullptr : units;
  }
  if (plan.form == LinearI4Plan::kMid) {
    if (!plan.wide) {
#define KERNEL(GJ, _) launch_mid<DT, 1, 2, GJ>(p, plan, planes, inv, ldp, s)
      ESM_I4_BY_GROUP(KERNEL, 0);
#undef KERNEL
    } else if constexpr (Elem<DT>::kPlanes == 1) {
      if (p.group == 64)
        launch_mid<DT, 2, 4, 2>(p, plan, planes, inv, ldp, s);
      else
        launch_mid<DT, 2, 4, 4>(p, plan, planes, inv, ldp, s);
    }
  } else {
    const unsigned grid =
        static_cast<unsigned>((p.M + kGemmM - 1) / kGemmM) * static_cast<unsigned>((p.N + kGemmN - 1) / kGemmN);
#define KERNEL(GJ, _) linear_i4_gemm_kernel<DT, GJ><<<grid, 256, 0, s>>>(p, planes, inv, ldp)
    ESM_I4_BY_GROUP(KERNEL, 0);
#undef KERNEL
  }
  return hipGetLastError();
}

}  // namespace

LinearI4Plan linear_i4_plan(const LinearI4Args& p, int type) {
  LinearI4Plan plan;
  const size_t tiles_n = (static_cast<size_t>(p.N) + kTileN - 1) / kTileN, cus = std::max(1, device_cus());
  // Rows that the kernels can read in place need no scratch, and no launch that
  // splits them (16 fp16 rows of 1,280 x 5,120 10.4 us split in the kernel, 7.0 read
  // in place). Splitting in every workgroup costs about 0.025 us a row and 128 inputs
  // on each CU, small tiles one more launch: 10 fp32 rows of 1,280 x 1,280 take 5.0
  // us split in the kernel (7.7 the other way), 13 of 1,280 x 5,120 13 (15), 8 of
  // 10,240 x 2,560 11 (14).
  const bool in_place = type == kTypeF16 && p.vec_a && p.K % kTileK == 0;
  const bool pairs = tiles_n >= 2 * cus && p.group != 32;  // two with four groups a tile spill
  const double row_cus = std::max(1.0, static_cast<double>(pairs ? tiles_n / 2 : tiles_n) / cus);
  const double tiles_us = (p.tiles_k + 7) / 8 + (0.5 + 0.12 * p.tiles_k) * (tiles_n / 2) / cus + 5.5;
  const double rows_us = 2.7 + 3.3e-3 * (p.group == 32 ? 1.7 : 1.0) * tiles_n * p.tiles_k / 8 +
                         0.025 * p.tiles_k * p.M * row_cus;
  if (p.M <= 4 || (p.M <= 16 && !in_place && rows_us <= tiles_us)) {
    plan.form = LinearI4Plan::kRows;
    plan.col_tiles = pairs ? 2 : 1;
    // As many waves as give each the same number of tiles, at most 10, and as many
    // of the waves' tiles at a time as keep the activations in 60 KB of LDS.
    const int rounds = (p.tiles_k + 9) / 10;
    plan.waves = (p.tiles_k + rounds - 1) / rounds;
    const int fit = static_cast<int>((size_t{60} << 10) / (p.M * ((type == kTypeF32 ? 512 : 256) + 4) + 16));
    plan.chunk = fit >= p.tiles_k ? p.tiles_k : fit / plan.waves * plan.waves;
    if (plan.chunk == 0) plan.chunk = plan.waves = std::max(1, fit);
    return plan;
  }
  const int ldp = in_place ? p.lda : p.tiles_k * kTileK;
  // The call's time on an idle device, in us, as measured over 17 to 4,096 rows of
  // 1,280 x 1,280, 3,840 x 1,280, 1,280 x 5,120, 2,560 x 2,560, 10,240 x 2,560 and
  // 2,560 x 10,240, the rows' split left out: small tiles 1 for each 128-input tile of
  // a wave and, as the CUs hold two or three, 0.5 (groups of 32: 0.75, turned round
  // 1.75) and 0.08 (two planes 0.12, groups of 32 0.03 more) per 128 inputs for each
  // of a CU's; wide ones 1.5 and 2.3 for each tile of a wave in each round of one
  // workgroup per CU; a GEMM workgroup 10 and 0.6 (two planes 0.97, groups of 32 0.5
  // more) per 64 inputs while it has a CU to itself, 1.4 times that where two share
  // one, and rounds of those (groups of 32 leave registers for one only). So 67 fp32
  // rows of 3,840 x 1,280 take small tiles (11 us, as a GEMM 40), 256 too (23, 42), 512
  // of 1,280 x 5,120 as well (40, 90) and 400 of 10,240 x 2,560 are a GEMM (76, in
  // small tiles 84); 301 fp16 rows of 1,280 x 5,120 take wide tiles (14, as a GEMM 57),
  // 256 of 2,560 x 10,240 small ones (40, wide 44).
  const bool two = type == kTypeF32, g32 = p.group == 32;
  auto tiles = [](int n, int by) { return (n + by - 1.0) / by; };
  const auto wgs = [&](int rows, int cols) { return std::floor(tiles(p.M, rows)) * std::floor(tiles(p.N, cols)); };
  const int iterations = (p.tiles_k + 7) / 8;
  const double gemm_wgs = wgs(kGemmM, kGemmN);
  const double of32 = g32 ? 1.0 : 0.0;
  const double small_each =
      0.5 + (in_place ? 1.25 : 0.25) * of32 + ((two ? 0.12 : 0.08) + 0.03 * of32) * p.tiles_k;
  const double small_us = iterations + small_each * wgs(16, 32) / cus;
  const double wide_us = two || g32 ? 1e30 : (1.5 + 2.3 * iterations) * std::ceil(wgs(32, 64) / cus);
  const double gemm_rounds = gemm_wgs <= cus ? 1.0
                             : g32           ? std::ceil(gemm_wgs / cus)
                                             : 1.4 * std::max(1.0, gemm_wgs / (2.0 * cus));
  const double gemm_us = (10.0 + ((two ? 0.97 : 0.6) + 0.5 * of32) * 2 * p.tiles_k) * gemm_rounds;
  // A GEMM tile's 64 rows are 32-bit offsets apart, and its grid is one number.
  const bool gemm_ok = ldp < (1 << 23) && gemm_wgs < 2e9;
  plan.wide = wide_us < small_us;
  plan.form = gemm_ok && gemm_us < std::min(small_us, wide_us) ? LinearI4Plan::kGemm : LinearI4Plan::kMid;
  plan.waves = (p.tiles_k + iterations - 1) / iterations;
  if (!in_place)
    plan.scratch_bytes =
        plane_elems(p.M, ldp) * (type == kTypeF32 ? 4 : 2) + static_cast<size_t>(p.M) * 4;
  return plan;
}

hipError_t launch_linear_i4(const LinearI4Args& p, const LinearI4Plan& plan, void* scratch, int type, hipStream_t s) {
  if (type == kTypeF32) return launch_typed<kTypeF32>(p, plan, scratch, s);
  if (type == kTypeF16) return launch_typed<kTypeF16>(p, plan, scratch, s);
  return launch_typed<kTypeBF16>(p, plan, scratch, s);
}

void linear_i4_layout(const uint8_t* packed, const float* scales, int N, int K, int group, uint32_t* w, float* s) {
  const int tiles_n = (N + kTileN - 1) / kTileN, tiles_k = (K + kTileK - 1) / kTileK;
  const int groups = (K + group - 1) / group;
  const size_t row_bytes = (static_cast<size_t>(K) + 1) / 2;
  for (int tn = 0; tn < tiles_n; ++tn)
    for (int kt = 0; kt < tiles_k; ++kt)
      for (int lane = 0; lane < 64; ++lane)
        for (int j = 0; j < 4; ++j) {
          const int n = tn * kTileN + lane % 16, k0 = kt * kTileK + 32 * j + 8 * (lane / 16);
          uint32_t v = 0;
          for (int i = 0; i < 8; ++i) {
            const int k = k0 + i;
            const uint32_t u = n < N && k < K ? (packed[n * row_bytes + k / 2] >> (4 * (k & 1))) & 15u : 8u;
            v |= u << (4 * (i / 2 + 4 * (i & 1)));
          }
          w[((static_cast<size_t>(tn) * tiles_k + kt) * 64 + lane) * 4 + j] = v;
        }
  for (int tn = 0; tn < tiles_n; ++tn)
    for (int g = 0; g < groups; ++g)
      for (int i = 0; i < kTileN; ++i) {
        const int n = tn * kTileN + i;
        s[(static_cast<size_t>(tn) * groups + g) * kTileN + i] = n < N ? scales[static_cast<size_t>(n) * groups + g] : 0.0f;
      }
}

}  // namespace esm_gfx950
