// Linears with 4-bit weights for gfx950: y = x W^T + bias, W[n, k] = code[n, k]
// * scale[n, k / group], codes in -8 .. 7, activations and outputs fp32, fp16 or
// bf16, sums in fp32.
//
// A code is an fp16 number as it stands, so the products run on fp16 MFMA with
// the weight operand exact: for fp16 activations directly, for bf16 ones (8
// significant bits) after a power of two per row and 128 inputs that brings the
// largest of them to [2^14, 2^15), and for fp32 ones as hi + lo fp16 parts (22
// significant bits) of the same scaled value, two MFMAs per product. A group's
// sum leaves the matrix cores before it is multiplied by its scale (and by the
// power of two's inverse): one fused multiply-add per output, group and row.
//
// Weights lie in tiles of 16 outputs x 128 inputs, 1 KB, in the order of the
// operand registers of v_mfma_f32_16x16x32_f16: lane n % 16 + 16 kq holds 16
// bytes, whose dword j has inputs 32 j + 8 kq .. + 8. Input 2 p of the eight is
// nibble p and input 2 p + 1 nibble p + 4, so that one and-or turns two codes
// into the fp16 pair 1024 + u (or 1024 + 16 u), and one packed add (fma) into
// the codes: nine instructions for eight weights.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace esm_gfx950 {

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kTileN = 16, kTileK = 128;

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

// The exponent e for which amax * 2^e lies in [2^14, 2^15) (amax finite;
// limited to what 2^e and 2^-e can be).
__device__ __forceinline__ int row_exponent(float amax) {
  return amax > 0.0f ? max(-120, min(120, 15 - __builtin_amdgcn_frexp_expf(amax))) : 0;
}

}  // namespace

// One workgroup: 16 MT rows x 16 NT outputs, its NW waves taking the 128-input
// tiles in turn and adding up through LDS. D = W x^T, so that a lane's outputs
// are four consecutive ones of the row l % 16 whose activations it also holds:
// the row's power of two needs no exchange, and a store is 16 bytes.
template <int DT, int MT, int NT, int GJ>  // GJ: 32-input steps of a group within a tile (1, 2 or 4)
__global__ __launch_bounds__(512) void linear_i4_rows_kernel(LinearI4Args p) {
  using T = typename Elem<DT>::T;
  constexpr int PL = Elem<DT>::kPlanes;
  extern __shared__ float red[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int lr = lane & 15, kq = lane >> 4;
  const int cols = (p.N + 16 * NT - 1) / (16 * NT);
  const int n0 = blockIdx.x % cols * (16 * NT), m0 = blockIdx.x / cols * (16 * MT);
  const int tiles_n = (p.N + kTileN - 1) / kTileN;
  const T* rows[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int m = m0 + 16 * mt + lr;
    rows[mt] = m < p.M ? static_cast<const T*>(p.A) + static_cast<size_t>(m) * p.lda : nullptr;
  }
  f32x4 total[NT][MT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) total[nt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int kt = wave; kt < p.tiles_k; kt += waves) {
    u32x4 w[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int tn = min(n0 / kTileN + nt, tiles_n - 1);
      w[nt] = reinterpret_cast<const u32x4*>(p.W)[(static_cast<size_t>(tn) * p.tiles_k + kt) * 64 + lane];
    }
    f16x8 a[MT][4][PL];
    float inv[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      T x[4][8];
#pragma unroll
      for (int j = 0; j < 4; ++j) load8<T>(rows[mt], kt * kTileK + 32 * j + 8 * kq, p.K, p.vec_a, x[j]);
      inv[mt] = 1.0f;
      if constexpr (DT == kTypeF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) __builtin_memcpy(&a[mt][j][0], x[j], 16);
      } else {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v = fabsf(static_cast<float>(x[j][i]));
            amax = fmaxf(amax, v < INFINITY ? v : 0.0f);
          }
        const LanePair s = lane_xor16(amax);
        amax = fmaxf(s.a, s.b);
        const LanePair t = lane_xor32(amax);
        amax = fmaxf(t.a, t.b);
        const int e = row_exponent(amax);
        const float mul = __builtin_amdgcn_ldexpf(1.0f, e);
        inv[mt] = __builtin_amdgcn_ldexpf(1.0f, -e);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v = static_cast<float>(x[j][i]) * mul;
            const _Float16 hi = static_cast<_Float16>(v);
            a[mt][j][0][i] = hi;
            if constexpr (PL == 2) a[mt][j][PL - 1][i] = static_cast<_Float16>(fabsf(v) < INFINITY ? v - static_cast<float>(hi) : 0.0f);
          }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int tn = min(n0 / kTileN + nt, tiles_n - 1);
      f32x4 acc[MT];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f16x8 wf = unpack_codes(w[nt][j]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          acc[mt] = mma(wf, a[mt][j][0], j % GJ == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[mt]);
          if constexpr (PL == 2) acc[mt] = mma(wf, a[mt][j][PL - 1], acc[mt]);
        }
        if ((j + 1) % GJ == 0) {
          const int g = min((kt * kTileK + 32 * j) / p.group, p.groups - 1);
          const f32x4 s = *reinterpret_cast<const f32x4*>(p.scales + (static_cast<size_t>(tn) * p.groups + g) * kTileN + 4 * kq);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              total[nt][mt][i] = __builtin_fmaf(acc[mt][i], s[i] * inv[mt], total[nt][mt][i]);
          }
        }
      }
    }
  }

  // The waves' sums meet in LDS and are added in the waves' order.
  f32x4* out4 = reinterpret_cast<f32x4*>(red);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) out4[(wave * NT * MT + nt * MT + mt) * 64 + lane] = total[nt][mt];
  __syncthreads();
  for (int u = wave; u < NT * MT; u += waves) {
    f32x4 sum = out4[u * 64 + lane];
    for (int w = 1; w < waves; ++w) sum += out4[(w * NT * MT + u) * 64 + lane];
    const int m = m0 + 16 * (u % MT) + lr, n = n0 + 16 * (u / MT) + 4 * kq;
    if (m >= p.M || n >= p.N) continue;
    T* c = static_cast<T*>(p.C) + static_cast<size_t>(m) * p.ldc + n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) c[i] = static_cast<T>(sum[i] + (p.bias ? p.bias[n + i] : 0.0f));
  }
}

// ------------------------------------------------------------- many rows
// Activations as the matrix cores take them, written once for every column tile:
// fp16 planes [planes][M][ldp] (hi, and lo for fp32), zeros past K, a row scaled
// by the power of two that brings its largest to [2^14, 2^15) (fp16 rows are
// taken as they are), the power's inverse in inv. One workgroup per row.
template <int DT>
__global__ __launch_bounds__(256) void linear_i4_split_kernel(LinearI4Args p, uint16_t* planes, float* inv, int ldp) {
  using T = typename Elem<DT>::T;
  __shared__ float part[4];
  const int m = blockIdx.x;
  const T* row = static_cast<const T*>(p.A) + static_cast<size_t>(m) * p.lda;
  uint16_t* hi = planes + static_cast<size_t>(m) * ldp;
  uint16_t* lo = hi + static_cast<size_t>(p.M) * ldp;
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
  } else {
    if (threadIdx.x == 0) inv[m] = 1.0f;
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
    *reinterpret_cast<f16x8*>(hi + k) = h;
    if constexpr (Elem<DT>::kPlanes == 2) *reinterpret_cast<f16x8*>(lo + k) = l;
  }
}

// 128 x 128 outputs per workgroup, 64 x 64 per wave on v_mfma_f32_32x32x16_f16:
// activations through LDS by direct loads, 64 inputs a stage, two stages; codes
// straight from global memory into the operand registers, the next 128 inputs'
// on their way. D has outputs across lanes: a group's scale is one register per
// 32 columns.
constexpr int kGemmM = 128, kGemmN = 128, kGemmK = 64;
template <int DT, int GJ>  // GJ: 32-input steps of a group within 128 inputs
__global__ __launch_bounds__(256) void linear_i4_gemm_kernel(LinearI4Args p, const uint16_t* planes, const float* inv,
                                                             int ldp) {
  using T = typename Elem<DT>::T;
  constexpr int PL = Elem<DT>::kPlanes;
  constexpr int kPlaneBytes = kGemmM * kGemmK * 2;
  typedef float f32x16 __attribute__((ext_vector_type(16)));
  __shared__ __align__(1024) uint8_t stage[2][PL * kPlaneBytes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ln = lane & 31, half = lane >> 5;
  int m0, n0;
  tile_origin_of(blockIdx.x, p.M, p.N, kGemmM, kGemmN, &m0, &n0);
  const int wm = wave >> 1, wn = wave & 1;

  // Direct loads: one instruction brings 8 rows of 64 inputs (1 KB); wave w loads
  // rows 32 w .. + 32. The 16-byte piece c of row r lies at c ^ (r % 8), so that
  // 32 rows' pieces fall on distinct banks.
  const uint32_t lds0 = lds_byte_addr(&stage[0][0]);
  uint32_t off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = wave * 32 + i * 8 + (lane >> 3), c = (lane & 7) ^ (lane >> 3);
    off[i] = static_cast<uint32_t>(min(r, p.M - 1 - m0)) * static_cast<uint32_t>(ldp * 2) + c * 16;
  }
  const size_t plane_elems = static_cast<size_t>(p.M) * ldp;
  auto load_stage = [&](int k0, int buf) {
#pragma unroll
    for (int pl = 0; pl < PL; ++pl) {
      const uint16_t* base = planes + pl * plane_elems + static_cast<size_t>(m0) * ldp + k0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        lds_dma16(base, off[i], lds0 + buf * (PL * kPlaneBytes) + pl * kPlaneBytes + (wave * 32 + i * 8) * 128);
    }
  };

  // Codes: for 16 inputs s of 128, lane (n, half) takes dword s / 2 of storage lane
  // n % 16 + 16 (2 (s % 2) + half).
  const int tiles_n = (p.N + kTileN - 1) / kTileN;
  const u32x4* wp[2];
  const float* sp[2];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    const int tn = min((n0 + wn * 64 + nt * 32) / kTileN + (ln >> 4), tiles_n - 1);
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
      const uint8_t* at = stage[h];
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const int step = h * 4 + st;  // of the 128 inputs' eight
        f16x8 wf[2];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) wf[nt] = unpack_codes(w[nt][step & 1][step >> 1]);
        const bool first = step % (2 * GJ) == 0;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const int r = wm * 64 + mt * 32 + ln;
          const uint8_t* a = at + r * 128 + (((2 * st + half) ^ (r & 7)) << 4);
          const f16x8 ah = *reinterpret_cast<const f16x8*>(a);
          f16x8 al;
          if constexpr (PL == 2) al = *reinterpret_cast<const f16x8*>(a + kPlaneBytes);
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            if (first) {
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[mt][nt][i] = 0.0f;
            }
            acc[mt][nt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, wf[nt], acc[mt][nt], 0, 0, 0);
            if constexpr (PL == 2) acc[mt][nt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, wf[nt], acc[mt][nt], 0, 0, 0);
          }
        }
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
      }
    }
  }

#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    const int n = n0 + wn * 64 + nt * 32 + ln;
    const float bias = p.bias && n < p.N ? p.bias[n] : 0.0f;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int m = m0 + wm * 64 + mt * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
        if (m < p.M && n < p.N)
          static_cast<T*>(p.C)[static_cast<size_t>(m) * p.ldc + n] =
              static_cast<T>(__builtin_fmaf(total[mt][nt][i], inv[m], bias));
      }
  }
}

namespace {

template <int DT, int MT, int NT>
hipError_t launch_rows(const LinearI4Args& p, hipStream_t s) {
  const int waves = std::min(NT * MT >= 16 ? 4 : 8, p.tiles_k);
  const unsigned grid =
      static_cast<unsigned>((p.N + 16 * NT - 1) / (16 * NT)) * ((p.M + 16 * MT - 1) / (16 * MT));
  const size_t lds = static_cast<size_t>(waves) * NT * MT * 1024;
  const dim3 block(64 * waves);
  if (p.group == 32)
    linear_i4_rows_kernel<DT, MT, NT, 1><<<grid, block, lds, s>>>(p);
  else if (p.group == 64)
    linear_i4_rows_kernel<DT, MT, NT, 2><<<grid, block, lds, s>>>(p);
  else
    linear_i4_rows_kernel<DT, MT, NT, 4><<<grid, block, lds, s>>>(p);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_gemm(const LinearI4Args& p, void* scratch, hipStream_t s) {
  const int ldp = p.tiles_k * kTileK;
  auto* planes = static_cast<uint16_t*>(scratch);
  auto* inv = reinterpret_cast<float*>(planes + static_cast<size_t>(Elem<DT>::kPlanes) * p.M * ldp);
  linear_i4_split_kernel<DT><<<p.M, 256, 0, s>>>(p, planes, inv, ldp);
  const unsigned grid =
      static_cast<unsigned>((p.M + kGemmM - 1) / kGemmM) * static_cast<unsigned>((p.N + kGemmN - 1) / kGemmN);
  if (p.group == 32)
    linear_i4_gemm_kernel<DT, 1><<<grid, 256, 0, s>>>(p, planes, inv, ldp);
  else if (p.group == 64)
    linear_i4_gemm_kernel<DT, 2><<<grid, 256, 0, s>>>(p, planes, inv, ldp);
  else
    linear_i4_gemm_kernel<DT, 4><<<grid, 256, 0, s>>>(p, planes, inv, ldp);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_typed(const LinearI4Args& p, const LinearI4Plan& plan, void* scratch, hipStream_t s) {
  if (plan.gemm) return launch_gemm<DT>(p, scratch, s);
  if (plan.row_tiles == 1) return launch_rows<DT, 1, 1>(p, s);
  if (plan.row_tiles == 2) return launch_rows<DT, 2, 2>(p, s);
  return launch_rows<DT, 4, 4>(p, s);
}

}  // namespace

LinearI4Plan linear_i4_plan(const LinearI4Args& p, int type) {
  LinearI4Plan plan;
  const int ldp = p.tiles_k * kTileK;
  // A tile's 128 rows are 32-bit offsets apart.
  plan.gemm = p.M > 256 && ldp < (1 << 23);
  plan.row_tiles = p.M <= 16 ? 1 : p.M <= 32 ? 2 : 4;
  if (plan.gemm)
    plan.scratch_bytes = static_cast<size_t>(p.M) * (static_cast<size_t>(ldp) * (type == kTypeF32 ? 4 : 2) + 4);
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
