// Block-sparse attention for gfx950: the mean key of every block of keys, the
// blocks whose mean scores highest for each query and head, and the attention
// over those blocks alone.
//
//   mean[j, h]    = (1 / n_j) sum of k[t, h] over block j's n_j keys, summed in
//                   64 bits, rounded to fp32
//   score[t,h,j]  = q[t, h] . mean[j, h / (heads / kv_heads)]
//   blocks[t, h]  = the `top` blocks of the query's sequence with the largest
//                   scores, ties to the lowest index, NaN as -inf; ascending,
//                   then -1
//   out[t, h]     = softmax over the listed blocks' keys of q . k, times v
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "kernels.hpp"

namespace esm_gfx950 {

namespace {

// Parts that the grouped attention has in flight between the pass that writes
// them and the one that joins them, some key heads at a time: no more than the
// 256 MB memory-side cache holds beside the keys (joining 138 MB took 24 us,
// 692 MB at once 175).
constexpr size_t kPartBytes = size_t{160} << 20;

// Division of 0 <= n < 2^31 by a launch's constant, in three instructions: with
// s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1, n / d is
// (floor(n m / 2^32) + n) / 2^s (Granlund and Montgomery, 1994).
struct Divisor {
  uint32_t mul = 0, shift = 0;
  Divisor() = default;
  explicit Divisor(int by) {
    while ((uint64_t{1} << shift) < static_cast<uint64_t>(by)) ++shift;
    mul = static_cast<uint32_t>(((uint64_t{1} << 32) * ((uint64_t{1} << shift) - by)) / by + 1);
  }
  __device__ __forceinline__ int operator()(int n) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), mul) + static_cast<uint32_t>(n)) >> shift);
  }
};

// The grouped attention's device scratch (attention, block by block).
struct GroupedWork {
  int token0 = 0, tokens = 0;  // the tokens in hand
  Divisor by_top, by_heads;
  int head_entries = 0;        // entries of a key head, counting or not
  int tile_entries = 0;        // most entries of a tile
  int group_heads = 0;         // key heads that are attended to together
  int group_tiles = 0;         // most tiles of such a group
  int* counts = nullptr;       // [cells] entries
  int* used = nullptr;         // [groups] tiles of a group (behind counts)
  int* first = nullptr;        // [cells] first entry in list
  int4* tiles = nullptr;       // [groups, group_tiles] (cell, first entry, entries, -), each key head's together
  int* place = nullptr;        // [entries] place in its cell, then in list; -1: does not count
  int* list = nullptr;         // [entries] by cell
  float2* part_ml = nullptr;   // [places of the heads in hand] maximum (base 2) and sum
  float* part_o = nullptr;     // [.., padded head_dim]; one entry more takes what belongs to none
};

template <int DT>
struct ElemOf;
template <>
struct ElemOf<kTypeF32> {
  using T = float;
};
template <>
struct ElemOf<kTypeF16> {
  using T = _Float16;
};
template <>
struct ElemOf<kTypeBF16> {
  using T = __bf16;
};

struct Seq {
  int k0, k1, b0, b1;
};

__device__ __forceinline__ int table_at(const SeqTable& t, const int* inl, int which, int i) {
  return t.dev ? t.dev[which * (t.batch + 1) + i] : inl[i];
}

// The sequence whose range of `which` (0 cu_q, 2 cb, 3 ct) holds x: the last one that
// starts at or before x (empty ranges hold nothing).
__device__ __forceinline__ int seq_of(const SeqTable& t, const int* inl, int which, int x) {
  int lo = 0, hi = t.batch;  // at(lo) <= x < at(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (table_at(t, inl, which, mid) <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ Seq seq_at(const SeqTable& t, int b) {
  return Seq{table_at(t, t.cu_k, 1, b), table_at(t, t.cu_k, 1, b + 1), table_at(t, t.cb, 2, b),
             table_at(t, t.cb, 2, b + 1)};
}

// Order-preserving key of a score: larger scores have larger keys, NaN counts
// as -inf and -0 as 0.
__device__ __forceinline__ uint64_t score_key(double s) {
  if (s != s) s = -INFINITY;
  const uint64_t u = __builtin_bit_cast(uint64_t, s + 0.0);
  return u >> 63 ? ~u : u | (uint64_t{1} << 63);
}

}  // namespace

// One workgroup per block and 64 16-byte column pieces: a lane has a piece, a wave
// every fourth key, eight loads in flight; the waves' 64-bit sums meet in LDS.
// Bound by the keys' bytes: 61,773 bf16 keys of 20 heads, 158 MB, in 27 us, at the
// rate of a large copy. (A thread per column, one element at a time, took 146.)
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void block_means_kernel(BlockAttnArgs p, SeqTable t) {
  using T = typename ElemOf<DT>::T;
  constexpr int E = 16 / sizeof(T);
  __shared__ double sums[3][E][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = blockIdx.x;
  const Seq s = seq_at(t, seq_of(t, t.cb, 2, j));
  const int t0 = s.k0 + (j - s.b0) * p.block_size, n = min(p.block_size, s.k1 - t0);
  const int cols = p.kv_heads * p.head_dim, col = (blockIdx.y * 64 + lane) * E;
  const bool mine = col < cols;
  const T* k = static_cast<const T*>(p.k) + static_cast<size_t>(t0) * p.ldkv + (mine ? col : 0);
  double sum[E];
#pragma unroll
  for (int i = 0; i < E; ++i) sum[i] = 0.0;
  for (int r0 = wave; r0 < n; r0 += 32) {
    T x[8][E];
#pragma unroll
    for (int u = 0; u < 8; ++u) {  // rows past the block's end read its last one, and do not count
      const T* at = k + static_cast<size_t>(min(r0 + 4 * u, n - 1)) * p.ldkv;
      if constexpr (VEC) {
        const uint4 v = *reinterpret_cast<const uint4*>(at);
        __builtin_memcpy(x[u], &v, 16);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[u][i] = at[i];
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (r0 + 4 * u < n) {
#pragma unroll
        for (int i = 0; i < E; ++i) sum[i] += static_cast<double>(static_cast<float>(x[u][i]));
      }
  }
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < E; ++i) sums[wave - 1][i][lane] = sum[i];
  }
  __syncthreads();
  if (wave > 0 || !mine) return;
  float* out = p.means_out + static_cast<size_t>(j) * cols + col;
#pragma unroll
  for (int i = 0; i < E; ++i)
    out[i] = static_cast<float>((((sum[i] + sums[0][i][lane]) + sums[1][i][lane]) + sums[2][i][lane]) / n);
}

namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));

// Order-preserving 32-bit key of an fp32 score, never 0.
__device__ __forceinline__ uint32_t score_key32(float s) {
  const uint32_t u = __float_as_uint(s + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// f over the lpr (4 .. 64) lanes that share a row, without a trip through LDS:
// quad permutations, then mirrors of 8 and 16 lanes (each half is uniform by
// then), then lane swaps.
template <class F>
__device__ __forceinline__ uint32_t row_reduce(uint32_t v, int lpr, F f) {
  v = f(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, true)));  // quad_perm [1, 0, 3, 2]
  v = f(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, true)));  // quad_perm [2, 3, 0, 1]
  if (lpr > 4) v = f(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true)));  // row_half_mirror
  if (lpr > 8) v = f(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true)));  // row_mirror
  if (lpr > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(r[0], r[1]);
  }
  if (lpr > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = f(r[0], r[1]);
  }
  return v;
}

// One wave: of the n 64-bit keys, the `want` largest (ties to the lowest index),
// handed to take(position, index, key) in ascending order of their indices.
// Their smallest is found bit by bit with counts by ballot.
template <class F>
__device__ __forceinline__ void take_largest(const uint64_t* keys, int n, int want, F take) {
  const int lane = threadIdx.x & 63;
  uint64_t thr = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t cand = thr | (uint64_t{1} << bit);
    int count = 0;
    for (int i = lane; i - lane < n; i += 64) count += __popcll(__ballot(i < n && keys[i] >= cand));
    if (count >= want) thr = cand;
  }
  int above = 0;
  for (int i = lane; i - lane < n; i += 64) above += __popcll(__ballot(i < n && keys[i] > thr));
  int equal = want - above, at = 0;
  for (int i = lane; i - lane < n; i += 64) {
    const uint64_t key = i < n ? keys[i] : 0;
    const bool eq = i < n && key == thr;
    const uint64_t eqs = __ballot(eq), below = (uint64_t{1} << lane) - 1;
    const bool mine = (i < n && key > thr) || (eq && static_cast<int>(__popcll(eqs & below)) < equal);
    equal -= min(equal, static_cast<int>(__popcll(eqs)));
    const uint64_t taken = __ballot(mine);
    if (mine) take(at + static_cast<int>(__popcll(taken & below)), i, key);
    at += __popcll(taken);
  }
}

__device__ __forceinline__ double score64(const float* q, const float* m, int dim) {
  double sum = 0.0;
  for (int d = 0; d < dim; ++d) sum += static_cast<double>(q[d]) * static_cast<double>(m[d]);
  return sum;
}

}  // namespace

// Rows of up to kSelBlocks blocks: a workgroup takes 16 `tiles` rows (queries of
// one key head, in token order) and scores them on fp64 MFMA, whose sums are far
// finer than the fp32 roundings that go to LDS. LPR lanes then share a row, each
// with up to 32 scores in registers, as integers spread evenly over the row's
// range, and find the top-th largest bit by bit, ending with the first threshold
// that exactly `top` of them reach (about as many steps as the row's range is
// powers of two of the gap there, two instructions per score each). Where that
// cannot tell the last ones apart, the row is settled with 64-bit scores.
//
// 7,930 queries of 20 heads over 21 to 65 blocks: 80 us, of it about 13 the fp64
// products; the threshold's steps on the VALU and their latency at 16 waves a CU are
// the rest. One wave per row with 64-bit scores summed lane by lane and a ballot per
// step took 2.2 ms.
constexpr int kSelBlocks = 960;  // a 16-row tile's keys fit 64 KB of LDS

template <int DT, int DH>
__global__ __launch_bounds__(1024) void select_rows_kernel(BlockAttnArgs p, SeqTable t, SelectPlan g) {
  using T = typename ElemOf<DT>::T;
  constexpr int kDims = DH / 4;  // dims per lane: kq * kDims .. + kDims
  extern __shared__ __align__(16) float scores[];
  __shared__ int unsettled[64];
  __shared__ float qs[kMaxHeadDim];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int hk = blockIdx.x % p.kv_heads, wg = blockIdx.x / p.kv_heads, each = p.heads / p.kv_heads;
  const int b = seq_of(t, t.ct, 3, wg);
  const int q0 = table_at(t, t.cu_q, 0, b), q1 = table_at(t, t.cu_q, 0, b + 1);
  const int b0 = table_at(t, t.cb, 2, b), nb = table_at(t, t.cb, 2, b + 1) - b0;
  const int row0 = (wg - table_at(t, t.ct, 3, b)) * 16 * g.tiles, rows = min((q1 - q0) * each - row0, 16 * g.tiles);
  const int want = min(p.top, nb);
  auto token_of = [&](int row) { return q0 + (row0 + row) / each; };
  auto head_of = [&](int row) { return hk * each + (row0 + row) % each; };
  for (int i = threadIdx.x; i < 64; i += blockDim.x) unsettled[i] = 0;

  // Scores: D = means . q^T, blocks down, queries across; lane (l % 16, kq) gives
  // block or query l % 16 the dims of kq, one per step.
  {
    const int lr = lane & 15, kq = lane >> 4, d0 = kq * kDims;
    const int row = wave % g.tiles * 16 + lr;
    double qd[kDims];
    const int rl = min(row, rows - 1);
    const T* q = static_cast<const T*>(p.q) + static_cast<size_t>(token_of(rl)) * p.ldq + head_of(rl) * p.head_dim;
    // Loads without conditions (each of which would be waited for on its own):
    // dims past the head read its last four, and count as zero.
    const int last = p.head_dim - 4;
    T qx[kDims];
#pragma unroll
    for (int i = 0; i < kDims; i += 4) {
      const T* at = q + min(d0 + i, last);
      if constexpr (DT == kTypeF32) {
        const f32x4 v = *reinterpret_cast<const f32x4u*>(at);
#pragma unroll
        for (int k = 0; k < 4; ++k) qx[i + k] = v[k];
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) qx[i + k] = at[k];
      }
    }
#pragma unroll
    for (int i = 0; i < kDims; ++i) qd[i] = d0 + i < p.head_dim ? static_cast<double>(static_cast<float>(qx[i])) : 0.0;
    const int step = waves / g.tiles * 16;
    float mf[kDims], next[kDims];
    auto load = [&](int bt, float (&to)[kDims]) {
      const float* m =
          p.means + (static_cast<size_t>(b0 + min(bt + lr, nb - 1)) * p.kv_heads + hk) * p.head_dim;
#pragma unroll
      for (int i = 0; i < kDims; i += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4u*>(m + min(d0 + i, last));
#pragma unroll
        for (int k = 0; k < 4; ++k) to[i + k] = d0 + i < p.head_dim ? v[k] : 0.0f;
      }
    };
    int bt = wave / g.tiles * 16;
    if (bt < nb) load(bt, next);
    for (; bt < nb; bt += step) {
#pragma unroll
      for (int i = 0; i < kDims; ++i) mf[i] = next[i];
      if (bt + step < nb) load(bt + step, next);
      f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int i = 0; i < kDims; ++i)
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64(static_cast<double>(mf[i]), qd[i], acc, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float s = static_cast<float>(acc[r]);
        scores[row * g.pitch + bt + 4 * r + kq] = s != s ? -INFINITY : s;
      }
    }
  }
  __syncthreads();

  // Thresholds: lane gl of a row's LPR has scores gl * per .. + per.
  const int lpr = g.lanes, gl = lane % lpr, per = ((nb + lpr - 1) / lpr + 3) & ~3;
  const int rows_per_wave = 64 / lpr;
  for (int u = wave * rows_per_wave; u < rows; u += waves * rows_per_wave) {
    const int row = u + lane / lpr;
    // A lane's scores, the number of which is uniform: four at a time.
    f32x4 s4[8];
    float most = -INFINITY, least = INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (4 * i < per) {
        const int at = gl * per + 4 * i;
        if (at < g.pitch) s4[i] = *reinterpret_cast<const f32x4*>(scores + min(row, rows - 1) * g.pitch + at);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (at + k < nb) {
            most = fmaxf(most, s4[i][k]);
            least = fminf(least, s4[i][k]);
          }
      }
    auto as_max = [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); };
    auto as_min = [](uint32_t a, uint32_t b) { return __float_as_uint(fminf(__uint_as_float(a), __uint_as_float(b))); };
    auto add = [](uint32_t a, uint32_t b) { return a + b; };
    most = __uint_as_float(row_reduce(__float_as_uint(most), lpr, as_max));
    least = __uint_as_float(row_reduce(__float_as_uint(least), lpr, as_min));
    // Keys 1 .. 2^30 over the row's range where that is finite, else the ordered
    // bits; 0 past the last block. Both keep the order of the scores.
    const float range = most - least;
    const bool even = range > 1e-28f && range < INFINITY;  // unit is finite
    const float unit = even ? 1073741696.0f / range : 0.0f;
    uint32_t k4[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (4 * i < per) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t key =
              even ? 1u + static_cast<uint32_t>((s4[i][k] - least) * unit) : score_key32(s4[i][k]);
          k4[i][k] = gl * per + 4 * i + k < nb ? key : 0;
        }
      }
    auto count_from = [&](uint32_t from) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (4 * i < per) {
#pragma unroll
          for (int k = 0; k < 4; ++k) n += k4[i][k] >= from;
        }
      return n;
    };
    uint32_t thr = want == nb ? 1 : 0;  // every block's key is at least 1
    bool settled = want == nb;
    for (int bit = __all(even) ? 30 : 31; bit >= 0 && !__all(settled); --bit) {
      const uint32_t cand = thr | (1u << bit);
      const int n = static_cast<int>(row_reduce(count_from(cand), lpr, add));
      if (!settled && n >= want) {
        thr = cand;
        settled = n == want;
      }
    }
    if (row >= rows) continue;
    int* out = p.blocks_out + (static_cast<size_t>(token_of(row)) * p.heads + head_of(row)) * p.top;
    for (int i = want + gl; i < p.top; i += lpr) out[i] = -1;
    if (!settled) {
      if (gl == 0) unsettled[row] = 1;
      continue;
    }
    const int mine = count_from(thr);
    int at = mine;
    for (int d = 1; d < lpr; d *= 2) {
      const int v = __shfl_up(at, d);
      at += gl >= d ? v : 0;
    }
    at -= mine;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (4 * i < per) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k4[i][k] >= thr) out[at++] = gl * per + 4 * i + k;
      }
  }

  // Rows whose last blocks are equal so far.
  __syncthreads();
  for (int row = 0; row < rows; ++row) {
    if (!unsettled[row]) continue;
    uint64_t* keys64 = reinterpret_cast<uint64_t*>(scores);  // every row's scores are done with
    const T* q = static_cast<const T*>(p.q) + static_cast<size_t>(token_of(row)) * p.ldq + head_of(row) * p.head_dim;
    for (int d = threadIdx.x; d < p.head_dim; d += blockDim.x) qs[d] = static_cast<float>(q[d]);
    __syncthreads();
    for (int j = threadIdx.x; j < nb; j += blockDim.x)
      keys64[j] = score_key(
          score64(qs, p.means + (static_cast<size_t>(b0 + j) * p.kv_heads + hk) * p.head_dim, p.head_dim));
    __syncthreads();
    if (wave == 0) {
      int* out = p.blocks_out + (static_cast<size_t>(token_of(row)) * p.heads + head_of(row)) * p.top;
      take_largest(keys64, nb, want, [&](int at, int i, uint64_t) { out[at] = i; });
    }
    __syncthreads();
  }
}

// Rows of any number of blocks, one wave per (query, head): 64-bit scores,
// kSelChunk blocks at a time behind the `top` kept from the chunks before.
constexpr int kSelChunk = 1024;
template <int DT>
__global__ __launch_bounds__(64) void select_blocks_kernel(BlockAttnArgs p, SeqTable t) {
  using T = typename ElemOf<DT>::T;
  __shared__ uint64_t keys[kSelChunk + kMaxTop];
  __shared__ int ids[kSelChunk + kMaxTop];
  __shared__ float qs[kMaxHeadDim];
  const int lane = threadIdx.x;
  const int row = blockIdx.x / p.heads, head = blockIdx.x % p.heads;
  const int hk = head / (p.heads / p.kv_heads);
  const Seq s = seq_at(t, seq_of(t, t.cu_q, 0, row));
  const int nb = s.b1 - s.b0;
  const T* q = static_cast<const T*>(p.q) + static_cast<size_t>(row) * p.ldq + head * p.head_dim;
  for (int d = lane; d < p.head_dim; d += 64) qs[d] = static_cast<float>(q[d]);
  __syncthreads();
  int kept = 0;
  for (int c0 = 0; c0 < nb; c0 += kSelChunk) {
    const int nc = min(kSelChunk, nb - c0);
    for (int i = lane; i < nc; i += 64) {
      keys[kept + i] = score_key(
          score64(qs, p.means + (static_cast<size_t>(s.b0 + c0 + i) * p.kv_heads + hk) * p.head_dim, p.head_dim));
      ids[kept + i] = c0 + i;
    }
    __syncthreads();
    // What is kept moves to the front, never past where it is read from.
    const int n = kept + nc;
    kept = min(p.top, n);
    take_largest(keys, n, kept, [&](int at, int i, uint64_t key) {
      const int id = ids[i];
      keys[at] = key;
      ids[at] = id;
    });
    __syncthreads();
  }
  int* out = p.blocks_out + (static_cast<size_t>(row) * p.heads + head) * p.top;
  for (int i = lane; i < p.top; i += 64) out[i] = i < kept ? ids[i] : -1;
}

namespace {

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ f32x4 mma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The exponent e for which amax * 2^e lies in [2^14, 2^15), where fp16 holds
// hi + lo parts to 22 bits down to 2^-39 of the largest; within -most .. most. Q
// and K are held to 60, so that the inverse of their scales' product is a normal
// number (a score's error is absolute: rows below 2^-45 only matter to keys above
// 2^20 and the other way round), V to 120.
__device__ __forceinline__ int scale_exponent(float amax, int most = 60) {
  return amax > 0.0f ? max(-most, min(most, 15 - __builtin_amdgcn_frexp_expf(amax))) : 0;
}

// Eight consecutive elements as fp32.
template <bool VEC, class T>
__device__ __forceinline__ void load8(const T* x, float (&out)[8]) {
  T v[8];
  if constexpr (VEC) {
    uint4 p[sizeof(T) / 2];
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) p[i] = reinterpret_cast<const uint4*>(x)[i];
    __builtin_memcpy(v, p, sizeof(p));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = static_cast<float>(v[i]);
}

// The largest of three, in one instruction (fmaxf quiets its operands first).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float max8(const float (&x)[8]) {  // of the magnitudes
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(m) : "v"(x[i]), "v"(x[i + 1]));
  return m;
}

// x * mul as fp16 hi parts, and lo parts where the type has two planes.
template <int PL>
__device__ __forceinline__ void split8(const float (&x)[8], float mul, uint4 (&out)[PL]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) split_pair(x[2 * j] * mul, x[2 * j + 1] * mul, &h[j], &l[j]);
  out[0] = make_uint4(h[0], h[1], h[2], h[3]);
  if constexpr (PL == 2) out[PL - 1] = make_uint4(l[0], l[1], l[2], l[3]);
}

// As lds_read_tr16 of the dense attention: lane s of 16 reads key s / 4 at
// positions 4 (s % 4) .. + 4 of a row-major tile, lane i receives position i of
// the four keys.
__device__ __forceinline__ f16x4 lds_read_tr16(const uint8_t* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)((__attribute__((address_space(3))) uint8_t*)p));
  return __builtin_bit_cast(f16x4, v);
}

__device__ __forceinline__ float group_max(float v) {  // over lanes ^ 16, ^ 32
  const LanePair a = lane_xor16(v);
  v = fmaxf(a.a, a.b);
  const LanePair b = lane_xor32(v);
  return fmaxf(b.a, b.b);
}
__device__ __forceinline__ float group_sum(float v) {
  const LanePair a = lane_xor16(v);
  v = a.a + a.b;
  const LanePair b = lane_xor32(v);
  return b.a + b.b;
}

}  // namespace

// ------------------------------------------------- attention, row by row
// Few rows: one workgroup per (query, head), a wave per listed block, joined in
// LDS. The 16-byte pieces of a key lie in LPK neighbouring lanes, 64 / LPK keys
// to a load. After the loads' products a butterfly over the lanes (each step
// hands half of the lane's values over) leaves every lane one key's score. Bound by
// the launch and three dependent trips to memory (list, keys, values): 3 queries of
// 20 heads, 16 blocks of 64 keys each, 11 us.
template <int DT, int DH, bool VEC>
__global__ __launch_bounds__(512) void attention_rows_kernel(BlockAttnArgs p, SeqTable t) {
  using T = typename ElemOf<DT>::T;
  constexpr int DPL = 16 / sizeof(T);        // dims per lane
  constexpr int LPK = DH / DPL;              // lanes per key
  constexpr int KPI = 64 / LPK;              // keys per load
  constexpr int IT = LPK < 16 ? LPK : 16;    // loads per round
  constexpr int KR = IT * KPI;               // keys per round: 64, or 32 with every score in two lanes
  __shared__ float part_o[8][DH], part_m[8], part_l[8];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int row = blockIdx.x / p.heads, head = blockIdx.x % p.heads;
  const int hk = head / (p.heads / p.kv_heads), dim = p.head_dim;
  const Seq s = seq_at(t, seq_of(t, t.cu_q, 0, row));
  const int d0 = lane % LPK * DPL, kl = lane / LPK;
  const int dl = d0 < dim ? d0 : 0;  // lanes past the head read its first dims, times zero
  const T* q = static_cast<const T*>(p.q) + static_cast<size_t>(row) * p.ldq + head * dim;
  const int* list = p.blocks + (static_cast<size_t>(row) * p.heads + head) * p.top;
  float qv[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) qv[i] = d0 < dim ? static_cast<float>(q[d0 + i]) * kLog2e : 0.0f;
  float m = -INFINITY, l = 0.0f, o[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) o[i] = 0.0f;

  for (int e = wave; e < p.top; e += waves) {
    const int j = list[e];
    if (j < 0 || j >= s.b1 - s.b0) continue;
    bool repeat = false;
    for (int i = lane; i < e; i += 64) repeat |= list[i] == j;
    if (__ballot(repeat)) continue;
    const int first = s.k0 + j * p.block_size, end = min(first + p.block_size, s.k1);
    for (int c = first; c < end; c += KR) {
      const int n = min(KR, end - c);
      uint4 kx[IT], vx[IT];
      // Rows past the block's end read its last key again, for a weight of zero.
      auto load = [&](const void* base, uint4 (&x)[IT]) {
        const T* at = static_cast<const T*>(base) + static_cast<size_t>(c) * p.ldkv + hk * dim;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const uint32_t off = static_cast<uint32_t>(min(i * KPI + kl, n - 1)) * static_cast<uint32_t>(p.ldkv) + dl;
          if constexpr (VEC) {
            x[i] = *reinterpret_cast<const uint4*>(at + off);
          } else {
            T y[DPL];
#pragma unroll
            for (int d = 0; d < DPL; ++d) y[d] = at[off + d];
            __builtin_memcpy(&x[i], y, 16);
          }
        }
      };
      load(p.k, kx);
      load(p.v, vx);
      float sc[IT];
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        T y[DPL];
        __builtin_memcpy(y, &kx[i], 16);
        sc[i] = 0.0f;
#pragma unroll
        for (int d = 0; d < DPL; ++d) sc[i] = __builtin_fmaf(qv[d], static_cast<float>(y[d]), sc[i]);
      }
      // After the steps over lane bits 1, 2, 4 .. this lane holds load `which`:
      // the bits of lane % IT reversed.
      int which = 0;
#pragma unroll
      for (int bit = 1, n2 = IT / 2; bit < IT; bit *= 2, n2 /= 2) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < n2; ++i) {
          const float keep = up ? sc[i + n2] : sc[i], give = up ? sc[i] : sc[i + n2];
          sc[i] = keep + __shfl_xor(give, bit);
        }
        which += up ? n2 : 0;
      }
      if constexpr (LPK > IT) sc[0] += __shfl_xor(sc[0], IT);
      const int key = which * KPI + kl;
      const float score = key < n ? sc[0] : -INFINITY;
      const float mn = fmaxf(m, wave_max(score));
      const float base = mn == -INFINITY ? 0.0f : mn;
      const float pr = exp2_raw(score - base), alpha = exp2_raw(m - base);
      l = l * alpha + wave_sum(LPK > IT && (lane & IT) ? 0.0f : pr);
      m = mn;
#pragma unroll
      for (int d = 0; d < DPL; ++d) o[d] *= alpha;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        // The lane of this group whose load is i: i's bits reversed.
        int from = 0;
#pragma unroll
        for (int bit = 1, n2 = IT / 2; bit < IT; bit *= 2, n2 /= 2) from |= i & n2 ? bit : 0;
        const float w = __shfl(pr, kl * LPK + from);
        T y[DPL];
        __builtin_memcpy(y, &vx[i], 16);
#pragma unroll
        for (int d = 0; d < DPL; ++d) o[d] = __builtin_fmaf(w, static_cast<float>(y[d]), o[d]);
      }
    }
  }
  // Sum over the lane groups' keys, then over the waves.
#pragma unroll
  for (int bit = LPK; bit < 64; bit *= 2)
#pragma unroll
    for (int d = 0; d < DPL; ++d) o[d] += __shfl_xor(o[d], bit);
  if (kl == 0)
#pragma unroll
    for (int d = 0; d < DPL; ++d) part_o[wave][d0 + d] = o[d];
  if (lane == 0) {
    part_m[wave] = m;
    part_l[wave] = l;
  }
  __syncthreads();
  float mm = -INFINITY;
  for (int w = 0; w < waves; ++w) mm = fmaxf(mm, part_m[w]);
  const float base = mm == -INFINITY ? 0.0f : mm;
  float sum = 0.0f;
  for (int w = 0; w < waves; ++w) sum += part_l[w] * exp2_raw(part_m[w] - base);
  for (int d = threadIdx.x; d < dim; d += blockDim.x) {
    float x = 0.0f;
    for (int w = 0; w < waves; ++w) x += part_o[w][d] * exp2_raw(part_m[w] - base);
    static_cast<T*>(p.out)[(static_cast<size_t>(row) * p.heads + head) * dim + d] =
        static_cast<T>(sum == 0.0f ? 0.0f : x / sum);
  }
}

// ----------------------------------------------- attention, block by block
// Many rows: the lists are turned round. Every cell (key head, block) gets the
// entries that list it, and a workgroup multiplies 512 of them with the cell's
// keys and values on the matrix cores, however few neighbours share a block;
// each entry's part (maximum, sum, weighted values) is written down, a
// workgroup's together, and a last pass gathers the parts of a row in the order
// of its list. So no result depends on the order in which a cell's entries were
// collected.
//
// An entry is (token - token0, head, list index) as one number; cells are
// numbered key head first.
constexpr int kCountThreads = 256, kCountPer = 16, kCountEntries = kCountThreads * kCountPer, kCountBlocks = 8192;
// A workgroup's entries: 512 where that fills the CUs twice, else 128.
constexpr int kTileEntries = 512, kSmallTileEntries = 128;

// The entries of one workgroup of the two list kernels: one head, and as many
// tokens as give kCountEntries entries (one token where it has more).
struct EntryRange {
  int head, hk, first, entries;
};
__device__ __forceinline__ EntryRange entry_range(const BlockAttnArgs& p, const GroupedWork& g) {
  const int per = kCountEntries / p.top, head = blockIdx.x % p.heads, first = blockIdx.x / p.heads * per;
  return EntryRange{head, head / (p.heads / p.kv_heads), first, min(per, g.tokens - first) * p.top};
}

// Counts the entries of each cell and gives each entry its place in it (-1: it
// does not count). A workgroup's counts meet in LDS first where the batch's
// blocks fit it, so that a cell sees one atomic per workgroup.
__global__ __launch_bounds__(kCountThreads) void count_entries_kernel(BlockAttnArgs p, SeqTable t, GroupedWork g) {
  __shared__ int hist[kCountBlocks];
  __shared__ int unsorted[kCountEntries];  // by token of the range
  const EntryRange r = entry_range(p, g);
  int* cells = g.counts + static_cast<size_t>(r.hk) * p.num_blocks;
  const bool lds = p.num_blocks <= kCountBlocks;
  // Every load first: entry u * 256 + thread of the range, and the one before it.
  int block[kCountPer], before[kCountPer], tok[kCountPer];
  const int* lists = p.blocks + (static_cast<size_t>(g.token0 + r.first) * p.heads + r.head) * p.top;
#pragma unroll
  for (int u = 0; u < kCountPer; ++u) {
    const int i = min(u * kCountThreads + static_cast<int>(threadIdx.x), r.entries - 1);
    tok[u] = g.by_top(i);
    const int e = i - tok[u] * p.top;
    const int* at = lists + static_cast<size_t>(tok[u]) * p.heads * p.top + e;
    block[u] = *at;
    before[u] = at[e > 0 ? -1 : 0];
  }
  for (int i = threadIdx.x; lds && i < p.num_blocks; i += kCountThreads) hist[i] = 0;
  for (int i = threadIdx.x, n = g.by_top(r.entries); i < n; i += kCountThreads) unsorted[i] = 0;
  __syncthreads();
  // A list that ascends and then ends in negatives, as the selection's do, has
  // no repeats.
#pragma unroll
  for (int u = 0; u < kCountPer; ++u) {
    const int i = u * kCountThreads + threadIdx.x;
    if (i >= r.entries) block[u] = -1;
    if (i - tok[u] * p.top > 0 && block[u] >= 0 && (before[u] < 0 || block[u] <= before[u])) unsorted[tok[u]] = 1;
  }
  __syncthreads();
  int place[kCountPer];
#pragma unroll
  for (int u = 0; u < kCountPer; ++u) {
    place[u] = -1;
    if (block[u] < 0) continue;
    const Seq s = seq_at(t, seq_of(t, t.cu_q, 0, g.token0 + r.first + tok[u]));
    bool counts = block[u] < s.b1 - s.b0;
    if (unsorted[tok[u]]) {
      const int* list = lists + static_cast<size_t>(tok[u]) * p.heads * p.top;
      const int e = u * kCountThreads + threadIdx.x - tok[u] * p.top;
      for (int k = 0; k < e; ++k) counts &= list[k] != block[u];
    }
    if (!counts) continue;
    block[u] += s.b0;
    place[u] = atomicAdd(lds ? &hist[block[u]] : &cells[block[u]], 1);
  }
  if (lds) {
    __syncthreads();
    for (int i = threadIdx.x; i < p.num_blocks; i += kCountThreads) {
      const int n = hist[i];
      if (n) hist[i] = atomicAdd(&cells[i], n);
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < kCountPer; ++u) {
    const int i = u * kCountThreads + threadIdx.x;
    if (i >= r.entries) continue;
    if (lds && place[u] >= 0) place[u] += hist[block[u]];
    g.place[(static_cast<size_t>(r.first + tok[u]) * p.heads + r.head) * p.top + (i - tok[u] * p.top)] = place[u];
  }
}

// One workgroup per key head: running sums over its cells' entries and tiles give
// every cell its stretch of the list and its tiles, behind the tiles of whichever
// heads of the group came before (nothing depends on their order). One thread per
// cell with atomics on the head's two totals took 29 us for 129 blocks of 20 heads.
constexpr int kPlaceThreads = 512;
__global__ __launch_bounds__(kPlaceThreads) void place_cells_kernel(BlockAttnArgs p, GroupedWork g) {
  __shared__ int sums[2][kPlaceThreads / 64];
  __shared__ int base;
  const int hk = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = hk / g.group_heads;
  auto cell_tiles = [&](int n) { return (n + g.tile_entries - 1) / g.tile_entries; };
  int mine = 0;
  for (int b = threadIdx.x; b < p.num_blocks; b += kPlaceThreads) mine += cell_tiles(g.counts[hk * p.num_blocks + b]);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) mine += __shfl_xor(mine, d);
  if (lane == 0) sums[0][wave] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int w = 0; w < kPlaceThreads / 64; ++w) n += sums[0][w];
    base = group * g.group_tiles + atomicAdd(&g.used[group], n);
  }
  __syncthreads();
  int at0 = hk * g.head_entries, tile0 = base;
  for (int c0 = 0; c0 < p.num_blocks; c0 += kPlaceThreads) {
    const int block = c0 + threadIdx.x, c = hk * p.num_blocks + block;
    const int n = block < p.num_blocks ? g.counts[c] : 0, tiles = cell_tiles(n);
    int n_to = n, tiles_to = tiles;  // sums over the wave's lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int a = __shfl_up(n_to, d), b = __shfl_up(tiles_to, d);
      n_to += lane >= d ? a : 0;
      tiles_to += lane >= d ? b : 0;
    }
    if (lane == 63) {
      sums[0][wave] = n_to;
      sums[1][wave] = tiles_to;
    }
    __syncthreads();
    int at = at0 + n_to - n, tile = tile0 + tiles_to - tiles;
#pragma unroll
    for (int w = 0; w < kPlaceThreads / 64; ++w) {
      at += w < wave ? sums[0][w] : 0;
      tile += w < wave ? sums[1][w] : 0;
      at0 += sums[0][w];
      tile0 += sums[1][w];
    }
    if (n) g.first[c] = at;
    for (int i = 0; i < tiles; ++i)
      g.tiles[tile + i] = make_int4(c, at + i * g.tile_entries, min(g.tile_entries, n - i * g.tile_entries), 0);
    __syncthreads();
  }
}

__global__ __launch_bounds__(kCountThreads) void scatter_entries_kernel(BlockAttnArgs p, SeqTable t, GroupedWork g) {
  const EntryRange r = entry_range(p, g);
  int at[kCountPer], place[kCountPer], block[kCountPer];
#pragma unroll
  for (int u = 0; u < kCountPer; ++u) {
    const int i = min(u * kCountThreads + static_cast<int>(threadIdx.x), r.entries - 1), tok = g.by_top(i);
    at[u] = ((r.first + tok) * p.heads + r.head) * p.top + (i - tok * p.top);
    place[u] = g.place[at[u]];
    block[u] = p.blocks[static_cast<size_t>(g.token0) * p.heads * p.top + at[u]] +
               seq_at(t, seq_of(t, t.cu_q, 0, g.token0 + r.first + tok)).b0;
  }
  int first[kCountPer];
#pragma unroll
  for (int u = 0; u < kCountPer; ++u) {
    if (u * kCountThreads + static_cast<int>(threadIdx.x) >= r.entries) place[u] = -1;
    first[u] = place[u] >= 0 ? g.first[r.hk * p.num_blocks + block[u]] : 0;
  }
#pragma unroll
  for (int u = 0; u < kCountPer; ++u)
    if (place[u] >= 0) {
      g.list[first[u] + place[u]] = at[u];
      g.place[at[u]] = first[u] + place[u];
    }
}

// One workgroup per tile of a cell's entries, 32 at a time to a wave.
// Keys and values come 64 at a time through LDS as fp16 (hi and lo planes for
// fp32 tensors), multiplied by powers of two that bring each 64 x dim tile's
// largest to [2^14, 2^15), and a row of q likewise: full precision whatever their
// magnitude. Blocks of at most 64 keys are staged once, and the waves then walk
// the tile's entries on their own, the next ones' queries on their way. S^T =
// K Q^T leaves a lane the scores of one query with keys 4 lg .. + 4 of every 16,
// which is the operand of O^T = V^T P^T as it stands.
//
// 8,195 queries of 20 heads, 16 blocks of 64 keys each, 43 GFLOP, run in five groups
// of heads: 65 us a group here (395 TFLOP/s of fp16 work, three products a fp32 one;
// softmax and splits on the VALU beside it, and 138 MB of parts written), 26 joining
// them, 40 for all the lists.
//
// ONE: no block is longer than 64 keys.
template <int DT, int DH, bool VEC, bool ONE>
__global__ __launch_bounds__(256) void attention_cells_kernel(BlockAttnArgs p, SeqTable t, GroupedWork g, int hk0,
                                                              int hk1) {
  using T = typename ElemOf<DT>::T;
  constexpr int PL = DT == kTypeF32 ? 2 : 1;
  constexpr int kPitch = DH * 2 + 16;  // 16 rows of 16 bytes fall on distinct banks
  constexpr int kPlane = 64 * kPitch;
  constexpr int kUnits = 64 * DH / 8 / 256;  // 8-element pieces per thread, of K and of V
  constexpr int KS = DH / 32;
  __shared__ __align__(16) uint8_t tile_k[PL * kPlane], tile_v[PL * kPlane];
  __shared__ float tile_max[2][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  // Workgroup i runs on XCD i % 8, and each XCD has its own L2: an XCD takes an
  // eighth of the tiles one after the other, two or three key heads' of 20, and
  // finds their queries in its L2.
  const int group = hk0 / g.group_heads, tiles = g.used[group], per = (tiles + 7) / 8;
  const int nth = blockIdx.x % 8 * per + blockIdx.x / 8;
  if (static_cast<int>(blockIdx.x / 8) >= per || nth >= tiles) return;
  const int4 tile = g.tiles[group * g.group_tiles + nth];
  const int hk = tile.x / p.num_blocks, block = tile.x - hk * p.num_blocks, dim = p.head_dim;
  const Seq s = seq_at(t, seq_of(t, t.cb, 2, block));
  const int key0 = s.k0 + (block - s.b0) * p.block_size, keys = min(p.block_size, s.k1 - key0);
  const int part0 = hk0 * g.head_entries, no_part = (hk1 - hk0) * g.head_entries;

  // Loads the 64 keys from key0 + c on, and their values, into LDS.
  int ke = 0, ve = 0;
  auto stage = [&](int c) {
    const int n = min(64, keys - c);
    float kx[kUnits][8], vx[kUnits][8];
    float kmax = 0.0f, vmax = 0.0f;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = u * 256 + threadIdx.x, key = unit / (DH / 8), d = unit % (DH / 8) * 8;
      const size_t at = static_cast<size_t>(key0 + c + key) * p.ldkv + hk * dim + d;
      if (key < n && d < dim) {
        load8<VEC>(static_cast<const T*>(p.k) + at, kx[u]);
        load8<VEC>(static_cast<const T*>(p.v) + at, vx[u]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) kx[u][i] = vx[u][i] = 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      kmax = fmaxf(kmax, max8(kx[u]));
      vmax = fmaxf(vmax, max8(vx[u]));
    }
    kmax = wave_max(kmax);
    vmax = wave_max(vmax);
    if (lane == 0) {
      tile_max[0][wave] = kmax;
      tile_max[1][wave] = vmax;
    }
    __syncthreads();  // also: the last 64 keys' reads are done
    ke = scale_exponent(fmaxf(fmaxf(tile_max[0][0], tile_max[0][1]), fmaxf(tile_max[0][2], tile_max[0][3])));
    ve = scale_exponent(fmaxf(fmaxf(tile_max[1][0], tile_max[1][1]), fmaxf(tile_max[1][2], tile_max[1][3])), 120);
    const float kmul = __builtin_amdgcn_ldexpf(1.0f, ke), vmul = __builtin_amdgcn_ldexpf(1.0f, ve);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = u * 256 + threadIdx.x, at = unit / (DH / 8) * kPitch + unit % (DH / 8) * 16;
      uint4 w[PL];
      split8<PL>(kx[u], kmul, w);
#pragma unroll
      for (int pl = 0; pl < PL; ++pl) *reinterpret_cast<uint4*>(tile_k + pl * kPlane + at) = w[pl];
      split8<PL>(vx[u], vmul, w);
#pragma unroll
      for (int pl = 0; pl < PL; ++pl) *reinterpret_cast<uint4*>(tile_v + pl * kPlane + at) = w[pl];
    }
    __syncthreads();
  };

  // This lane's two queries of the 128 entries from i0 on.
  int entry[2], next_entry[2];
  float qx[2][KS][8];
  auto list_at = [&](int i0, int (&to)[2]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = i0 + wave * 32 + r * 16 + lr, e = g.list[tile.y + min(i, tile.z - 1)];
      to[r] = i < tile.z ? e : -1;
    }
  };
  // Loads and stores without conditions, so that a wait for the next queries
  // counts the stores behind them instead of waiting for those too: lanes without
  // an entry read the first query and write past the last part, and dims past the
  // head read its first ones (the keys are zero there).
  auto load_q = [&](const int (&of)[2]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g.by_top(max(of[r], 0)), tok = g.by_heads(row), head = row - tok * p.heads;
      const T* q = static_cast<const T*>(p.q) + static_cast<size_t>(g.token0 + tok) * p.ldq + head * dim;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = ks * 32 + lg * 8;
        load8<VEC>(q + (d < dim ? d : 0), qx[r][ks]);
      }
    }
  };
  list_at(0, entry);
  load_q(entry);
  list_at(128, next_entry);
  if (ONE) stage(0);

  for (int i0 = 0; i0 < tile.z; i0 += 128) {
    const bool active = i0 + wave * 32 < tile.z;
    if (ONE && !active) break;  // no more barriers, and later entries are none of this wave's
    f16x8 qf[2][KS][PL];
    int qe[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float amax = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) amax = fmaxf(amax, max8(qx[r][ks]));
      qe[r] = scale_exponent(group_max(amax));
      const float mul = __builtin_amdgcn_ldexpf(1.0f, qe[r]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint4 w[PL];
        split8<PL>(qx[r][ks], mul, w);
#pragma unroll
        for (int pl = 0; pl < PL; ++pl) qf[r][ks][pl] = __builtin_bit_cast(f16x8, w[pl]);
      }
    }
    const int now[2] = {entry[0], entry[1]};
    entry[0] = next_entry[0];
    entry[1] = next_entry[1];
    load_q(entry);
    list_at(i0 + 256, next_entry);

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    f32x4 o[2][DH / 16];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int db = 0; db < DH / 16; ++db) o[r][db] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int c = 0; c < (ONE ? 1 : keys); c += 64) {
      const int n = min(64, keys - c);
      if constexpr (!ONE) {
        stage(c);
        if (!active) continue;
      }
      f32x4 sc[4][2];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
        for (int r = 0; r < 2; ++r) sc[kb][r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint8_t* at = tile_k + (kb * 16 + lr) * kPitch + (ks * 4 + lg) * 16;
          const f16x8 kh = *reinterpret_cast<const f16x8*>(at);
#pragma unroll
          for (int r = 0; r < 2; ++r) sc[kb][r] = mma16(kh, qf[r][ks][0], sc[kb][r]);
          if constexpr (PL == 2) {
            const f16x8 kl = *reinterpret_cast<const f16x8*>(at + kPlane);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              sc[kb][r] = mma16(kl, qf[r][ks][0], sc[kb][r]);
              sc[kb][r] = mma16(kh, qf[r][ks][PL - 1], sc[kb][r]);
            }
          }
        }
      }
      if (n < 64) {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (kb * 16 + lg * 4 + i >= n) sc[kb][r][i] = -INFINITY;
      }
      // Softmax in base 2: the scores' maximum first, then one fused step and an
      // exponential per score.
      f16x8 pf[2][2][PL];
      float alpha[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float unit = __builtin_amdgcn_ldexpf(kLog2e, -(qe[r] + ke));
        float mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          mx = max3(sc[kb][r][0], sc[kb][r][1], mx);
          mx = max3(sc[kb][r][2], sc[kb][r][3], mx);
        }
        const float mn = fmaxf(m[r], group_max(mx) * unit);
        const float base = mn == -INFINITY ? 0.0f : mn;
        alpha[r] = exp2_raw(m[r] - base);
        m[r] = mn;
        float sum = 0.0f;
#pragma unroll
        for (int kp = 0; kp < 2; ++kp) {
          float pr[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            pr[i] = exp2_raw(__builtin_fmaf(sc[2 * kp + (i >> 2)][r][i & 3], unit, -base));
            sum += pr[i];
          }
          uint4 w[PL];
          split8<PL>(pr, 1.0f, w);
#pragma unroll
          for (int pl = 0; pl < PL; ++pl) pf[r][kp][pl] = __builtin_bit_cast(f16x8, w[pl]);
        }
        l[r] = __builtin_fmaf(l[r], alpha[r], sum);
      }
      const float vunit = __builtin_amdgcn_ldexpf(1.0f, -ve);
#pragma unroll
      for (int db = 0; db < DH / 16; ++db) {
        f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int kp = 0; kp < 2; ++kp) {
          const uint8_t* at = tile_v + (kp * 32 + lg * 4 + (lr >> 2)) * kPitch + db * 32 + (lr & 3) * 8;
          auto frag = [&](const uint8_t* x) {
            const f16x4 a = lds_read_tr16(x), b = lds_read_tr16(x + 16 * kPitch);
            return f16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
          };
          const f16x8 vh = frag(at);
#pragma unroll
          for (int r = 0; r < 2; ++r) acc[r] = mma16(vh, pf[r][kp][0], acc[r]);
          if constexpr (PL == 2) {
            const f16x8 vl = frag(at + kPlane);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              acc[r] = mma16(vl, pf[r][kp][0], acc[r]);
              acc[r] = mma16(vh, pf[r][kp][PL - 1], acc[r]);
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            o[r][db][i] = ONE ? acc[r][i] * vunit : __builtin_fmaf(o[r][db][i], alpha[r], acc[r][i] * vunit);
      }
    }

#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float sum = group_sum(l[r]);
      const int i = i0 + wave * 32 + r * 16 + lr;
      const size_t at = now[r] < 0 ? no_part : tile.y + i - part0;
      g.part_ml[at] = make_float2(m[r], sum);  // the same from all four lanes
#pragma unroll
      for (int db = 0; db < DH / 16; ++db)
        *reinterpret_cast<f32x4*>(g.part_o + at * DH + db * 16 + lg * 4) = o[r][db];
    }
  }
}

// One row's parts, joined in the order of its list by GL lanes: a lane weighs
// one entry of every GL and sums four dims of all of them.
template <int DT, int GL>
__global__ __launch_bounds__(256) void join_entries_kernel(BlockAttnArgs p, GroupedWork g, int hk0, int hk1) {
  using T = typename ElemOf<DT>::T;
  const int each = p.heads / p.kv_heads, chunk_heads = (hk1 - hk0) * each;
  const int gl = threadIdx.x % GL;
  const size_t rows = static_cast<size_t>(g.tokens) * chunk_heads;
  const size_t mine = (blockIdx.x * size_t{256} + threadIdx.x) / GL;
  const size_t row = mine < rows ? mine : rows - 1;  // lanes past the end keep the shuffles whole
  const int d = gl * 4, dl = d < p.head_dim ? d : 0;
  const size_t tok = row / chunk_heads;
  const int head = static_cast<int>(row - tok * chunk_heads) + hk0 * each;
  const int* place = g.place + (tok * p.heads + head) * p.top;
  const int part0 = hk0 * g.head_entries;
  constexpr int kStride = GL * 4 < 32 ? 32 : GL * 4;  // the parts' padded head_dim
  const float* o = g.part_o + dl;
  float m = -INFINITY, sum = 0.0f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int e0 = 0; e0 < p.top; e0 += GL) {
    const int n = min(GL, p.top - e0);
    const int at = gl < n ? place[e0 + gl] - part0 : -1;
    const bool counts = at >= 0;
    const float2 v = counts ? g.part_ml[at] : make_float2(-INFINITY, 0.0f);
    float mx = v.x;
#pragma unroll
    for (int b = 1; b < GL; b *= 2) mx = fmaxf(mx, __shfl_xor(mx, b));
    const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.0f : mn;
    const float alpha = exp2_raw(m - base), w = counts ? exp2_raw(v.x - base) : -1.0f;
    float part = counts ? v.y * w : 0.0f;
#pragma unroll
    for (int b = 1; b < GL; b *= 2) part += __shfl_xor(part, b);
    sum = __builtin_fmaf(sum, alpha, part);
    m = mn;
    x *= alpha;
    for (int e = 0; e < n; e += 8) {
      f32x4 y[8];
      float ws[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        ws[k] = __shfl(w, min(e + k, n - 1), GL);
        if (e + k >= n) ws[k] = -1.0f;
        const int from = __shfl(at, min(e + k, n - 1), GL);
        y[k] = *reinterpret_cast<const f32x4*>(o + static_cast<size_t>(max(from, 0)) * kStride);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ws[k] != -1.0f ? __builtin_fmaf(y[k][i], ws[k], x[i]) : x[i];
    }
  }
  if (mine >= rows || d >= p.head_dim) return;
  T* out = static_cast<T*>(p.out) + ((static_cast<size_t>(g.token0) + tok) * p.heads + head) * p.head_dim + d;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = static_cast<T>(sum == 0.0f ? 0.0f : x[i] / sum);
}

namespace {

template <int DT>
hipError_t launch_means_typed(const BlockAttnArgs& p, const SeqTable& t, hipStream_t s) {
  constexpr int kCols = 64 * 16 / sizeof(typename ElemOf<DT>::T);  // of a workgroup
  const dim3 grid(p.num_blocks, (p.kv_heads * p.head_dim + kCols - 1) / kCols);
  if (p.vec_kv)
    block_means_kernel<DT, true><<<grid, 256, 0, s>>>(p, t);
  else
    block_means_kernel<DT, false><<<grid, 256, 0, s>>>(p, t);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_block_means(const BlockAttnArgs& p, const SeqTable& t, int type, hipStream_t s) {
  if (type == kTypeF32) return launch_means_typed<kTypeF32>(p, t, s);
  if (type == kTypeF16) return launch_means_typed<kTypeF16>(p, t, s);
  return launch_means_typed<kTypeBF16>(p, t, s);
}

namespace {

template <int DT>
hipError_t launch_select_typed(const BlockAttnArgs& p, const SeqTable& t, const SelectPlan& g, hipStream_t s) {
  if (!g.tiles) {
    select_blocks_kernel<DT><<<static_cast<unsigned>(p.rows) * p.heads, 64, 0, s>>>(p, t);
    return hipGetLastError();
  }
  const unsigned grid = static_cast<unsigned>(g.workgroups) * p.kv_heads, block = 64 * g.waves;
  const size_t lds = static_cast<size_t>(16) * g.tiles * g.pitch * 4;
  if (p.head_dim <= 16)
    select_rows_kernel<DT, 16><<<grid, block, lds, s>>>(p, t, g);
  else if (p.head_dim <= 32)
    select_rows_kernel<DT, 32><<<grid, block, lds, s>>>(p, t, g);
  else if (p.head_dim <= 64)
    select_rows_kernel<DT, 64><<<grid, block, lds, s>>>(p, t, g);
  else
    select_rows_kernel<DT, 128><<<grid, block, lds, s>>>(p, t, g);
  return hipGetLastError();
}

}  // namespace

SelectPlan select_blocks_plan(const BlockAttnArgs& p, const int* cu_q, int batch, int max_blocks) {
  SelectPlan g;
  if (max_blocks > kSelBlocks) return g;
  while (g.lanes * 32 < max_blocks) g.lanes *= 2;
  g.pitch = (max_blocks + 15) / 16 * 16 + 4;  // 16 rows of 4 scores fall on distinct banks
  // Four tiles, one to a wave, where that leaves a workgroup for every CU and
  // LDS for two of them on one; else one tile for all waves.
  const size_t many = static_cast<size_t>(p.rows) * p.heads / 64;
  g.tiles = many >= static_cast<size_t>(device_cus()) && g.pitch <= 256 ? 4 : 1;
  g.waves = g.tiles == 4 ? 4 : std::max(4, std::min(16, (max_blocks + 15) / 16));
  size_t n = 0;
  for (int b = 0; b < batch; ++b) n += select_workgroups(p, g, cu_q[b + 1] - cu_q[b]);
  g.workgroups = static_cast<int>(n);  // at most one per (query, head)
  return g;
}

int select_workgroups(const BlockAttnArgs& p, const SelectPlan& g, int queries) {
  const size_t rows = static_cast<size_t>(queries) * (p.heads / p.kv_heads);
  return g.tiles ? static_cast<int>((rows + 16 * g.tiles - 1) / (16 * g.tiles)) : 0;
}

hipError_t launch_select_blocks(const BlockAttnArgs& p, const SeqTable& t, const SelectPlan& g, int type,
                                hipStream_t s) {
  if (type == kTypeF32) return launch_select_typed<kTypeF32>(p, t, g, s);
  if (type == kTypeF16) return launch_select_typed<kTypeF16>(p, t, g, s);
  return launch_select_typed<kTypeBF16>(p, t, g, s);
}

namespace {

size_t up256(size_t v) { return (v + 255) & ~size_t{255}; }

int padded_dim(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

// The grouped form's scratch for a plan, laid out from base on.
GroupedWork grouped_layout(const BlockAttnArgs& p, const BlockAttnPlan& plan, char* base, size_t* bytes) {
  const size_t cells = static_cast<size_t>(p.num_blocks) * p.kv_heads;
  const size_t entries = static_cast<size_t>(plan.tokens) * p.heads * p.top, head_entries = entries / p.kv_heads;
  const size_t head_tiles = head_entries / plan.tile_entries + std::min<size_t>(p.num_blocks, head_entries);
  const int groups = (p.kv_heads + plan.kv_heads - 1) / plan.kv_heads;
  const size_t parts = head_entries * plan.kv_heads;
  GroupedWork g;
  size_t at = 0;
  auto take = [&](size_t n) {
    char* q = base ? base + at : nullptr;
    at += up256(n);
    return q;
  };
  g.by_top = Divisor(p.top);
  g.by_heads = Divisor(p.heads);
  g.head_entries = static_cast<int>(head_entries);
  g.tile_entries = plan.tile_entries;
  g.group_heads = plan.kv_heads;
  g.group_tiles = static_cast<int>(head_tiles * plan.kv_heads);
  g.counts = reinterpret_cast<int*>(take((cells + groups) * 4));
  g.used = g.counts ? g.counts + cells : nullptr;
  g.first = reinterpret_cast<int*>(take(cells * 4));
  g.tiles = reinterpret_cast<int4*>(take(head_tiles * plan.kv_heads * groups * 16));
  g.place = reinterpret_cast<int*>(take(entries * 4));
  g.list = reinterpret_cast<int*>(take(entries * 4));
  g.part_ml = reinterpret_cast<float2*>(take((parts + 1) * 8));
  g.part_o = reinterpret_cast<float*>(take((parts + 1) * padded_dim(p.head_dim) * 4));
  *bytes = at;
  return g;
}

template <int DT, int DH>
hipError_t launch_attention_rows(const BlockAttnArgs& p, const SeqTable& t, const BlockAttnPlan& plan, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(p.rows) * p.heads, block = 64 * plan.waves;
  if (p.vec_kv)
    attention_rows_kernel<DT, DH, true><<<grid, block, 0, s>>>(p, t);
  else
    attention_rows_kernel<DT, DH, false><<<grid, block, 0, s>>>(p, t);
  return hipGetLastError();
}

template <int DT>
void launch_join(const BlockAttnArgs& p, const GroupedWork& g, int h0, int h1, size_t rows, hipStream_t s) {
  const auto grid = [&](int lanes) { return static_cast<unsigned>((rows * lanes + 255) / 256); };
  if (p.head_dim <= 16)
    join_entries_kernel<DT, 4><<<grid(4), 256, 0, s>>>(p, g, h0, h1);
  else if (p.head_dim <= 32)
    join_entries_kernel<DT, 8><<<grid(8), 256, 0, s>>>(p, g, h0, h1);
  else if (p.head_dim <= 64)
    join_entries_kernel<DT, 16><<<grid(16), 256, 0, s>>>(p, g, h0, h1);
  else
    join_entries_kernel<DT, 32><<<grid(32), 256, 0, s>>>(p, g, h0, h1);
}

template <int DT, int DH>
hipError_t launch_attention_cells(const BlockAttnArgs& p, const SeqTable& t, const BlockAttnPlan& plan, void* scratch,
                                  hipStream_t s) {
  size_t bytes = 0;
  GroupedWork g = grouped_layout(p, plan, static_cast<char*>(scratch), &bytes);
  const int cells = p.num_blocks * p.kv_heads, each = p.heads / p.kv_heads;
  for (int t0 = 0; t0 < p.rows; t0 += plan.tokens) {
    g.token0 = t0;
    g.tokens = p.rows - t0 < plan.tokens ? p.rows - t0 : plan.tokens;
    const int groups = (p.kv_heads + g.group_heads - 1) / g.group_heads;
    // Integer zeros for counts and used.
    const hipError_t e = launch_fill_f32(reinterpret_cast<float*>(g.counts), cells + groups, 0.0f, s);
    if (e != hipSuccess) return e;
    const int per = kCountEntries / p.top;
    const unsigned ranges = static_cast<unsigned>((g.tokens + per - 1) / per) * p.heads;
    count_entries_kernel<<<ranges, kCountThreads, 0, s>>>(p, t, g);
    place_cells_kernel<<<p.kv_heads, kPlaceThreads, 0, s>>>(p, g);
    scatter_entries_kernel<<<ranges, kCountThreads, 0, s>>>(p, t, g);
    for (int h0 = 0; h0 < p.kv_heads; h0 += g.group_heads) {
      const int h1 = std::min(h0 + g.group_heads, p.kv_heads);
      const unsigned grid = static_cast<unsigned>(g.group_tiles + 7) / 8 * 8;
      const bool vec = p.vec_kv && p.vec_q;
      if (p.block_size <= 64)
        vec ? attention_cells_kernel<DT, DH, true, true><<<grid, 256, 0, s>>>(p, t, g, h0, h1)
            : attention_cells_kernel<DT, DH, false, true><<<grid, 256, 0, s>>>(p, t, g, h0, h1);
      else
        vec ? attention_cells_kernel<DT, DH, true, false><<<grid, 256, 0, s>>>(p, t, g, h0, h1)
            : attention_cells_kernel<DT, DH, false, false><<<grid, 256, 0, s>>>(p, t, g, h0, h1);
      launch_join<DT>(p, g, h0, h1, static_cast<size_t>(g.tokens) * (h1 - h0) * each, s);
    }
    const hipError_t done = hipGetLastError();
    if (done != hipSuccess) return done;
  }
  return hipSuccess;
}

template <int DT>
hipError_t launch_attention_typed(const BlockAttnArgs& p, const SeqTable& t, const BlockAttnPlan& plan, void* scratch,
                                  hipStream_t s) {
  if (!plan.grouped)
    return p.head_dim <= 32   ? launch_attention_rows<DT, 32>(p, t, plan, s)
           : p.head_dim <= 64 ? launch_attention_rows<DT, 64>(p, t, plan, s)
                              : launch_attention_rows<DT, 128>(p, t, plan, s);
  return p.head_dim <= 32   ? launch_attention_cells<DT, 32>(p, t, plan, scratch, s)
         : p.head_dim <= 64 ? launch_attention_cells<DT, 64>(p, t, plan, scratch, s)
                            : launch_attention_cells<DT, 128>(p, t, plan, scratch, s);
}

}  // namespace

BlockAttnPlan attention_blocks_plan(const BlockAttnArgs& p, const int* cu_q, const int* cu_k, int batch, int type) {
  BlockAttnPlan plan;
  const size_t cells = static_cast<size_t>(p.num_blocks) * p.kv_heads;
  const size_t row_entries = static_cast<size_t>(p.heads) * p.top;  // of a token
  // The entries that can count, and their keys.
  double entries = 0.0, keys = 0.0;
  int most = 0;
  for (int b = 0; b < batch; ++b) {
    const int n = cu_k[b + 1] - cu_k[b], blocks = n > 0 ? (n - 1) / p.block_size + 1 : 0;
    const double rows = static_cast<double>(cu_q[b + 1] - cu_q[b]) * p.heads;
    entries += rows * std::min(p.top, blocks);
    keys += rows * std::min<double>(static_cast<double>(p.top) * p.block_size, n);
    most = std::max(most, std::min(p.top, blocks));
  }
  plan.waves = std::max(1, std::min(8, most));
  if (cells == 0 || cells > 0x3fffffff || entries == 0.0) return plan;
  // Both forms' time in us, as measured over 4 to 768 queries of 8 to 40 heads: row
  // by row 5 and every entry's keys and values, of 64 keys at least, at 9.5 TB/s
  // (from L2); block by block 24 (six launches), 7.5e-3 for every 32 KB that a
  // workgroup stages and 0.25e-3 for every 32 KB of keys and values that an entry
  // meets in LDS. 20 heads of 64, fp32: 64 queries over their one block each 9 and
  // 25, 192 over 3 57 and 28, 16 over 16 of 250 45 and 49, 100 over 16 of 250 182
  // and 65; half precision: 128 over 2 14 and 26.
  const double row_bytes = p.head_dim * 2.0 * (type == kTypeF32 ? 4 : 2);  // a key and its value
  const double unit = keys / entries * row_bytes / 32768.0;
  const double hit = cells * (1.0 - std::exp(-entries / cells));
  const double rows_us = 5.0 + entries * std::max(keys / entries, 64.0) * row_bytes / 9.5e6;
  const double cells_us = 24.0 + (hit + entries / kTileEntries) * 7.5e-3 * unit + entries * 0.25e-3 * unit;
  plan.grouped = cells_us < rows_us;
  if (!plan.grouped) return plan;
  plan.tile_entries = hit + entries / kTileEntries >= 2.0 * device_cus() ? kTileEntries : kSmallTileEntries;
  // Entry numbers are 32-bit, and lists of 2^26 entries take half a gigabyte.
  plan.tokens = static_cast<int>(std::min<size_t>(p.rows, std::max<size_t>(1, (size_t{1} << 26) / row_entries)));
  const size_t head_bytes =
      static_cast<size_t>(plan.tokens) * (p.heads / p.kv_heads) * p.top * (padded_dim(p.head_dim) * 4 + 8);
  plan.kv_heads = static_cast<int>(std::min<size_t>(p.kv_heads, std::max<size_t>(1, kPartBytes / head_bytes)));
  grouped_layout(p, plan, nullptr, &plan.scratch_bytes);
  return plan;
}

hipError_t launch_attention_blocks(const BlockAttnArgs& p, const SeqTable& t, const BlockAttnPlan& plan, void* scratch,
                                   int type, hipStream_t s) {
  if (type == kTypeF32) return launch_attention_typed<kTypeF32>(p, t, plan, scratch, s);
  if (type == kTypeF16) return launch_attention_typed<kTypeF16>(p, t, plan, scratch, s);
  return launch_attention_typed<kTypeBF16>(p, t, plan, scratch, s);
}

}  // namespace esm_gfx950
