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

#include "common.hpp"
#include "kernels.hpp"

namespace esm_gfx950 {

namespace {

// Parts of the grouped attention that are in flight between the pass that
// writes them and the one that joins them: what the 256 MB memory-side cache
// holds beside the keys.
constexpr size_t kPartBytes = size_t{128} << 20;

// The grouped attention's device scratch (attention, block by block).
struct GroupedWork {
  int token0 = 0, tokens = 0;  // the tokens in hand
  int* counts = nullptr;       // [cells] entries
  int* first = nullptr;        // [cells] first entry in list
  int* cell_tile = nullptr;    // [cells + 1] first tile
  int4* tiles = nullptr;       // (cell, first entry, entries, -)
  int* place = nullptr;        // [entries] place in its cell, -1: does not count
  int* list = nullptr;         // [entries] by cell
  float2* part_ml = nullptr;   // [entries of the heads in hand] maximum (base 2) and sum
  float* part_o = nullptr;     // [.., head_dim]
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
  int q0, k0, k1, b0, b1;
};

__device__ __forceinline__ int table_at(const SeqTable& t, const int* inl, int which, int i) {
  return t.dev ? t.dev[which * (t.batch + 1) + i] : inl[i];
}

// The sequence whose range of `which` (0 cu_q, 2 cb) holds x: the last one that
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
  return Seq{table_at(t, t.cu_q, 0, b), table_at(t, t.cu_k, 1, b), table_at(t, t.cu_k, 1, b + 1),
             table_at(t, t.cb, 2, b), table_at(t, t.cb, 2, b + 1)};
}

// Order-preserving key of a score: larger scores have larger keys, NaN counts
// as -inf and -0 as 0.
__device__ __forceinline__ uint64_t score_key(double s) {
  if (s != s) s = -INFINITY;
  const uint64_t u = __builtin_bit_cast(uint64_t, s + 0.0);
  return u >> 63 ? ~u : u | (uint64_t{1} << 63);
}

}  // namespace

// One workgroup per block: a thread sums a column of the block's keys.
template <int DT>
__global__ __launch_bounds__(256) void block_means_kernel(BlockAttnArgs p, SeqTable t) {
  using T = typename ElemOf<DT>::T;
  const int j = blockIdx.x;
  const Seq s = seq_at(t, seq_of(t, t.cb, 2, j));
  const int t0 = s.k0 + (j - s.b0) * p.block_size, n = min(p.block_size, s.k1 - t0);
  const int cols = p.kv_heads * p.head_dim;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    const T* k = static_cast<const T*>(p.k) + static_cast<size_t>(t0) * p.ldkv + c;
    double sum = 0.0;
    for (int r = 0; r < n; ++r) sum += static_cast<double>(static_cast<float>(k[static_cast<size_t>(r) * p.ldkv]));
    p.means_out[static_cast<size_t>(j) * cols + c] = static_cast<float>(sum / n);
  }
}

// One wave per (query, head). Scores in 64 bits, kept as order-preserving keys
// in LDS, kSelChunk blocks at a time behind the `top` kept from the chunks
// before; the top-th largest key is found bit by bit with counts by ballot, and
// what is above it (and equal to it, lowest index first) stays in order.
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
      const float* m = p.means + (static_cast<size_t>(s.b0 + c0 + i) * p.kv_heads + hk) * p.head_dim;
      double sum = 0.0;
      for (int d = 0; d < p.head_dim; ++d) sum += static_cast<double>(qs[d]) * static_cast<double>(m[d]);
      keys[kept + i] = score_key(sum);
      ids[kept + i] = c0 + i;
    }
    __syncthreads();
    const int n = kept + nc, want = min(p.top, n);
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
      const int id = i < n ? ids[i] : 0;
      const bool eq = i < n && key == thr;
      const uint64_t eqs = __ballot(eq), below = (uint64_t{1} << lane) - 1;
      const bool take = (i < n && key > thr) || (eq && static_cast<int>(__popcll(eqs & below)) < equal);
      equal -= min(equal, static_cast<int>(__popcll(eqs)));
      const uint64_t takes = __ballot(take);
      __syncthreads();
      if (take) {
        keys[at + __popcll(takes & below)] = key;
        ids[at + __popcll(takes & below)] = id;
      }
      __syncthreads();
      at += __popcll(takes);
    }
    kept = want;
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
// hi + lo parts to 22 bits and everything 2^-39 above the largest.
__device__ __forceinline__ int scale_exponent(float amax) {
  return amax > 0.0f ? max(-120, min(120, 15 - __builtin_amdgcn_frexp_expf(amax))) : 0;
}

// Eight consecutive elements as fp32.
template <class T>
__device__ __forceinline__ void load8(const T* x, bool vec, float (&out)[8]) {
  T v[8];
  if (vec) {
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

__device__ __forceinline__ float max8(const float (&x)[8]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
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

// Whether entry e of a row's list counts: a block of the sequence, and no
// repeat of an earlier entry.
__device__ __forceinline__ bool entry_counts(const int* list, int e, int nb) {
  const int j = list[e];
  if (j < 0 || j >= nb) return false;
  for (int i = 0; i < e; ++i)
    if (list[i] == j) return false;
  return true;
}

}  // namespace

// ------------------------------------------------- attention, row by row
// Few rows: one workgroup per (query, head), a wave per listed block, joined in
// LDS. The 16-byte pieces of a key lie in LPK neighbouring lanes, 64 / LPK keys
// to a load. After the loads' products a butterfly over the lanes (each step
// hands half of the lane's values over) leaves every lane one key's score.
template <int DT, int DH>
__global__ __launch_bounds__(512) void attention_rows_kernel(BlockAttnArgs p, SeqTable t) {
  using T = typename ElemOf<DT>::T;
  constexpr int DPL = 16 / sizeof(T);        // dims per lane
  constexpr int LPK = DH / DPL;              // lanes per key
  constexpr int KPI = 64 / LPK;              // keys per load
  constexpr int IT = LPK < 16 ? LPK : 16;    // loads per round
  constexpr int KR = IT * KPI;               // keys per round: 64, or 32 with every score in two lanes
  __shared__ float part_o[8][DH], part_m[8], part_l[8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
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
          if (p.vec_kv) {
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
// entries that list it, and a workgroup multiplies 128 of them with the cell's
// keys and values on the matrix cores, however few neighbours share a block;
// each entry's part (maximum, sum, weighted values) is written down by entry,
// and a last pass joins the entries of a row in the order of its list. So no
// result depends on the order in which a cell's entries were collected.
//
// An entry is (token - token0, head, list index) as one number; cells are
// numbered key head first.
constexpr int kCountThreads = 256, kCountEntries = 4096, kCountBlocks = 8192;
constexpr int kTileEntries = 128;

// Counts the entries of each cell and gives each entry its place in it (-1: it
// does not count). One workgroup per head and as many tokens as give
// kCountEntries entries; their counts meet in LDS first where the batch's blocks
// fit it, so that a cell sees one atomic per workgroup.
__global__ __launch_bounds__(kCountThreads) void count_entries_kernel(BlockAttnArgs p, SeqTable t, GroupedWork g,
                                                                      int tokens_per_group) {
  __shared__ int hist[kCountBlocks];
  const int head = blockIdx.x % p.heads, first = blockIdx.x / p.heads * tokens_per_group;
  const int tokens = min(tokens_per_group, g.tokens - first);
  const int hk = head / (p.heads / p.kv_heads);
  int* cells = g.counts + static_cast<size_t>(hk) * p.num_blocks;
  const bool lds = p.num_blocks <= kCountBlocks;
  if (lds) {
    for (int i = threadIdx.x; i < p.num_blocks; i += kCountThreads) hist[i] = 0;
    __syncthreads();
  }
  const int entries = tokens * p.top;
  for (int i = threadIdx.x; i < entries; i += kCountThreads) {
    const int tok = first + i / p.top, e = i % p.top;
    const Seq s = seq_at(t, seq_of(t, t.cu_q, 0, g.token0 + tok));
    const int* list = p.blocks + (static_cast<size_t>(g.token0 + tok) * p.heads + head) * p.top;
    int place = -1;
    if (entry_counts(list, e, s.b1 - s.b0)) {
      const int j = s.b0 + list[e];
      place = lds ? atomicAdd(&hist[j], 1) : atomicAdd(&cells[j], 1);
    }
    g.place[(static_cast<size_t>(tok) * p.heads + head) * p.top + e] = place;
  }
  if (!lds) return;
  __syncthreads();
  for (int i = threadIdx.x; i < p.num_blocks; i += kCountThreads) {
    const int n = hist[i];
    if (n) hist[i] = atomicAdd(&cells[i], n);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < entries; i += kCountThreads) {
    const int tok = first + i / p.top, e = i % p.top;
    const size_t at = (static_cast<size_t>(tok) * p.heads + head) * p.top + e;
    const int place = g.place[at];
    if (place < 0) continue;
    const Seq s = seq_at(t, seq_of(t, t.cu_q, 0, g.token0 + tok));
    const int j = s.b0 + p.blocks[(static_cast<size_t>(g.token0 + tok) * p.heads + head) * p.top + e];
    g.place[at] = place + hist[j];
  }
}

// One workgroup: the cells' first entries and tiles (running sums over the
// counts), and the tiles themselves.
constexpr int kScanThreads = 1024;
__global__ __launch_bounds__(kScanThreads) void scan_cells_kernel(GroupedWork g, int cells) {
  __shared__ int sums[2][kScanThreads];
  const int per = (cells + kScanThreads - 1) / kScanThreads;
  const int c0 = min(cells, static_cast<int>(threadIdx.x) * per), c1 = min(cells, c0 + per);
  int entries = 0, tiles = 0;
  for (int c = c0; c < c1; ++c) {
    entries += g.counts[c];
    tiles += (g.counts[c] + kTileEntries - 1) / kTileEntries;
  }
  sums[0][threadIdx.x] = entries;
  sums[1][threadIdx.x] = tiles;
  __syncthreads();
  for (int d = 1; d < kScanThreads; d *= 2) {
    const int a = threadIdx.x >= d ? sums[0][threadIdx.x - d] : 0, b = threadIdx.x >= d ? sums[1][threadIdx.x - d] : 0;
    __syncthreads();
    sums[0][threadIdx.x] += a;
    sums[1][threadIdx.x] += b;
    __syncthreads();
  }
  int at = sums[0][threadIdx.x] - entries, tile = sums[1][threadIdx.x] - tiles;
  for (int c = c0; c < c1; ++c) {
    const int n = g.counts[c];
    g.first[c] = at;
    g.cell_tile[c] = tile;
    for (int i = 0; i < n; i += kTileEntries) g.tiles[tile++] = make_int4(c, at + i, min(kTileEntries, n - i), 0);
    at += n;
  }
  if (threadIdx.x == kScanThreads - 1) g.cell_tile[cells] = tile;
}

__global__ __launch_bounds__(256) void scatter_entries_kernel(BlockAttnArgs p, SeqTable t, GroupedWork g) {
  const size_t n = static_cast<size_t>(g.tokens) * p.heads * p.top;
  for (size_t i = blockIdx.x * size_t{256} + threadIdx.x; i < n; i += size_t{256} * gridDim.x) {
    const int place = g.place[i];
    if (place < 0) continue;
    const int row = static_cast<int>(i / p.top), tok = row / p.heads, hk = row % p.heads / (p.heads / p.kv_heads);
    const Seq s = seq_at(t, seq_of(t, t.cu_q, 0, g.token0 + tok));
    const int j = s.b0 + p.blocks[static_cast<size_t>(g.token0) * p.heads * p.top + i];
    g.list[g.first[hk * p.num_blocks + j] + place] = static_cast<int>(i);
  }
}

// One workgroup per tile of 128 entries, 32 to a wave. Keys and values come 64
// at a time through LDS as fp16 (hi and lo planes for fp32 tensors), multiplied
// by powers of two that bring each 64 x dim tile's largest to [2^14, 2^15), and
// a row of q likewise: full precision at every magnitude. S^T = K Q^T leaves a
// lane the scores of one query with keys 4 lg .. + 4 of every 16, which is the
// operand of O^T = V^T P^T as it stands.
template <int DT, int DH>
__global__ __launch_bounds__(256) void attention_cells_kernel(BlockAttnArgs p, SeqTable t, GroupedWork g, int hk0,
                                                              int hk1) {
  using T = typename ElemOf<DT>::T;
  constexpr int PL = DT == kTypeF32 ? 2 : 1;
  constexpr int kPitch = DH * 2 + 16;  // 16 rows of 16 bytes fall on distinct banks
  constexpr int kPlane = 64 * kPitch;
  constexpr int kUnits = 64 * DH / 8 / 256;  // 8-element pieces per thread, of K and of V
  __shared__ __align__(16) uint8_t tile_k[PL * kPlane], tile_v[PL * kPlane];
  __shared__ float tile_max[2][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lr = lane & 15, lg = lane >> 4;
  const int tile0 = g.cell_tile[hk0 * p.num_blocks], tile_end = g.cell_tile[hk1 * p.num_blocks];
  if (tile0 + static_cast<int>(blockIdx.x) >= tile_end) return;
  const int4 tile = g.tiles[tile0 + blockIdx.x];
  const int hk = tile.x / p.num_blocks, block = tile.x % p.num_blocks, dim = p.head_dim;
  const Seq s = seq_at(t, seq_of(t, t.cb, 2, block));
  const int key0 = s.k0 + (block - s.b0) * p.block_size, keys = min(p.block_size, s.k1 - key0);
  const int each = p.heads / p.kv_heads, chunk_heads = (hk1 - hk0) * each;

  // This lane's queries.
  int entry[2], head[2], tok[2];
  f16x8 qf[2][DH / 32][PL];
  int qe[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = wave * 32 + r * 16 + lr;
    entry[r] = i < tile.z ? g.list[tile.y + i] : -1;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = max(entry[r], 0) / p.top;
    tok[r] = row / p.heads;
    head[r] = row % p.heads;
    const T* q = static_cast<const T*>(p.q) + static_cast<size_t>(g.token0 + tok[r]) * p.ldq + head[r] * dim;
    float x[DH / 32][8];
    float amax = 0.0f;
#pragma unroll
    for (int ks = 0; ks < DH / 32; ++ks) {
      const int d = ks * 32 + lg * 8;
      if (entry[r] >= 0 && d < dim) {
        load8<T>(q + d, p.vec_q, x[ks]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[ks][i] = 0.0f;
      }
      amax = fmaxf(amax, max8(x[ks]));
    }
    qe[r] = scale_exponent(group_max(amax));
    const float mul = __builtin_amdgcn_ldexpf(1.0f, qe[r]);
#pragma unroll
    for (int ks = 0; ks < DH / 32; ++ks) {
      uint4 w[PL];
      split8<PL>(x[ks], mul, w);
#pragma unroll
      for (int pl = 0; pl < PL; ++pl) qf[r][ks][pl] = __builtin_bit_cast(f16x8, w[pl]);
    }
  }
  const bool active = wave * 32 < tile.z;

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  f32x4 o[2][DH / 16];
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int db = 0; db < DH / 16; ++db) o[r][db] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int c = 0; c < keys; c += 64) {
    const int n = min(64, keys - c);
    float kx[kUnits][8], vx[kUnits][8];
    float kmax = 0.0f, vmax = 0.0f;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = u * 256 + threadIdx.x, key = unit / (DH / 8), d = unit % (DH / 8) * 8;
      const size_t at = static_cast<size_t>(key0 + c + key) * p.ldkv + hk * dim + d;
      if (key < n && d < dim) {
        load8<T>(static_cast<const T*>(p.k) + at, p.vec_kv, kx[u]);
        load8<T>(static_cast<const T*>(p.v) + at, p.vec_kv, vx[u]);
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
    __syncthreads();  // also: the last tile's reads are done
    const int ke = scale_exponent(fmaxf(fmaxf(tile_max[0][0], tile_max[0][1]), fmaxf(tile_max[0][2], tile_max[0][3])));
    const int ve = scale_exponent(fmaxf(fmaxf(tile_max[1][0], tile_max[1][1]), fmaxf(tile_max[1][2], tile_max[1][3])));
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
    if (!active) continue;

    f32x4 sc[4][2];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
      for (int r = 0; r < 2; ++r) sc[kb][r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < DH / 32; ++ks) {
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
    f16x8 pf[2][2][PL];
    float alpha[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = __builtin_amdgcn_ldexpf(sc[kb][r][i], -(qe[r] + ke)) * kLog2e;
          sc[kb][r][i] = kb * 16 + lg * 4 + i < n ? v : -INFINITY;
          mx = fmaxf(mx, sc[kb][r][i]);
        }
      const float mn = fmaxf(m[r], group_max(mx));
      const float base = mn == -INFINITY ? 0.0f : mn;
      alpha[r] = exp2_raw(m[r] - base);
      m[r] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int kp = 0; kp < 2; ++kp) {
        float pr[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pr[i] = exp2_raw(sc[2 * kp + (i >> 2)][r][i & 3] - base);
          sum += pr[i];
        }
        uint4 w[PL];
        split8<PL>(pr, 1.0f, w);
#pragma unroll
        for (int pl = 0; pl < PL; ++pl) pf[r][kp][pl] = __builtin_bit_cast(f16x8, w[pl]);
      }
      l[r] = __builtin_fmaf(l[r], alpha[r], sum);
    }
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
          o[r][db][i] = __builtin_fmaf(o[r][db][i], alpha[r], __builtin_amdgcn_ldexpf(acc[r][i], -ve));
    }
  }

#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float sum = group_sum(l[r]);
    if (entry[r] < 0) continue;
    const size_t at =
        (static_cast<size_t>(tok[r]) * chunk_heads + head[r] - hk0 * each) * p.top + entry[r] % p.top;
    if (lg == 0) g.part_ml[at] = make_float2(m[r], sum);
#pragma unroll
    for (int db = 0; db < DH / 16; ++db)
      if (db * 16 + lg * 4 < dim) *reinterpret_cast<f32x4*>(g.part_o + at * dim + db * 16 + lg * 4) = o[r][db];
  }
}

// One row's parts, dim / 4 lanes to an entry, joined in the order of its list.
template <int DT>
__global__ __launch_bounds__(256) void join_entries_kernel(BlockAttnArgs p, GroupedWork g, int hk0, int hk1) {
  using T = typename ElemOf<DT>::T;
  const int each = p.heads / p.kv_heads, chunk_heads = (hk1 - hk0) * each;
  const int quads = p.head_dim / 4;
  const size_t i = blockIdx.x * size_t{256} + threadIdx.x;
  const size_t row = i / quads;
  if (row >= static_cast<size_t>(g.tokens) * chunk_heads) return;
  const int d = static_cast<int>(i % quads) * 4;
  const size_t tok = row / chunk_heads;
  const int head = static_cast<int>(row % chunk_heads) + hk0 * each;
  const int* place = g.place + (tok * p.heads + head) * p.top;
  const float2* ml = g.part_ml + row * p.top;
  const float* o = g.part_o + row * p.top * p.head_dim + d;
  float m = -INFINITY;
  for (int e = 0; e < p.top; ++e)
    if (place[e] >= 0) m = fmaxf(m, ml[e].x);
  const float base = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int e = 0; e < p.top; ++e) {
    if (place[e] < 0) continue;
    const float w = exp2_raw(ml[e].x - base);
    sum = __builtin_fmaf(ml[e].y, w, sum);
    const f32x4 v = *reinterpret_cast<const f32x4*>(o + static_cast<size_t>(e) * p.head_dim);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __builtin_fmaf(v[k], w, x[k]);
  }
  T* out = static_cast<T*>(p.out) + ((static_cast<size_t>(g.token0) + tok) * p.heads + head) * p.head_dim + d;
#pragma unroll
  for (int k = 0; k < 4; ++k) out[k] = static_cast<T>(sum == 0.0f ? 0.0f : x[k] / sum);
}

hipError_t launch_block_means(const BlockAttnArgs& p, const SeqTable& t, int type, hipStream_t s) {
  if (type == kTypeF32)
    block_means_kernel<kTypeF32><<<p.num_blocks, 256, 0, s>>>(p, t);
  else if (type == kTypeF16)
    block_means_kernel<kTypeF16><<<p.num_blocks, 256, 0, s>>>(p, t);
  else
    block_means_kernel<kTypeBF16><<<p.num_blocks, 256, 0, s>>>(p, t);
  return hipGetLastError();
}

hipError_t launch_select_blocks(const BlockAttnArgs& p, const SeqTable& t, int type, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(p.rows) * p.heads;
  if (type == kTypeF32)
    select_blocks_kernel<kTypeF32><<<grid, 64, 0, s>>>(p, t);
  else if (type == kTypeF16)
    select_blocks_kernel<kTypeF16><<<grid, 64, 0, s>>>(p, t);
  else
    select_blocks_kernel<kTypeBF16><<<grid, 64, 0, s>>>(p, t);
  return hipGetLastError();
}

namespace {

size_t up256(size_t v) { return (v + 255) & ~size_t{255}; }

// The grouped form's scratch for a plan, laid out from base on.
GroupedWork grouped_layout(const BlockAttnArgs& p, const BlockAttnPlan& plan, char* base, size_t* bytes) {
  const size_t cells = static_cast<size_t>(p.num_blocks) * p.kv_heads;
  const size_t entries = static_cast<size_t>(plan.tokens) * p.heads * p.top;
  const size_t parts = static_cast<size_t>(plan.tokens) * plan.kv_heads * (p.heads / p.kv_heads) * p.top;
  GroupedWork g;
  size_t at = 0;
  auto take = [&](size_t n) {
    char* q = base ? base + at : nullptr;
    at += up256(n);
    return q;
  };
  g.counts = reinterpret_cast<int*>(take(cells * 4));
  g.first = reinterpret_cast<int*>(take(cells * 4));
  g.cell_tile = reinterpret_cast<int*>(take((cells + 1) * 4));
  g.tiles = reinterpret_cast<int4*>(take((entries / kTileEntries + cells + 1) * 16));
  g.place = reinterpret_cast<int*>(take(entries * 4));
  g.list = reinterpret_cast<int*>(take(entries * 4));
  g.part_ml = reinterpret_cast<float2*>(take(parts * 8));
  g.part_o = reinterpret_cast<float*>(take(parts * p.head_dim * 4));
  *bytes = at;
  return g;
}

template <int DT, int DH>
hipError_t launch_attention_rows(const BlockAttnArgs& p, const SeqTable& t, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(p.rows) * p.heads;
  attention_rows_kernel<DT, DH><<<grid, 64 * (p.top < 8 ? p.top : 8), 0, s>>>(p, t);
  return hipGetLastError();
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
    const size_t entries = static_cast<size_t>(g.tokens) * p.heads * p.top;
    hipError_t e = launch_fill_f32(reinterpret_cast<float*>(g.counts), cells, 0.0f, s);  // integer zeros
    if (e != hipSuccess) return e;
    const int per = kCountEntries / p.top;
    const unsigned groups = static_cast<unsigned>((g.tokens + per - 1) / per) * p.heads;
    count_entries_kernel<<<groups, kCountThreads, 0, s>>>(p, t, g, per);
    scan_cells_kernel<<<1, kScanThreads, 0, s>>>(g, cells);
    const unsigned sgrid = static_cast<unsigned>(entries / 256 + 1 < 16384 ? entries / 256 + 1 : 16384);
    scatter_entries_kernel<<<sgrid, 256, 0, s>>>(p, t, g);
    for (int h0 = 0; h0 < p.kv_heads; h0 += plan.kv_heads) {
      const int h1 = h0 + plan.kv_heads < p.kv_heads ? h0 + plan.kv_heads : p.kv_heads;
      const size_t rows = static_cast<size_t>(g.tokens) * (h1 - h0) * each;
      const size_t tiles = rows * p.top / kTileEntries + static_cast<size_t>(h1 - h0) * p.num_blocks;
      attention_cells_kernel<DT, DH><<<static_cast<unsigned>(tiles), 256, 0, s>>>(p, t, g, h0, h1);
      join_entries_kernel<DT><<<static_cast<unsigned>((rows * (p.head_dim / 4) + 255) / 256), 256, 0, s>>>(p, g, h0, h1);
    }
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int DT>
hipError_t launch_attention_typed(const BlockAttnArgs& p, const SeqTable& t, const BlockAttnPlan& plan, void* scratch,
                                  hipStream_t s) {
  if (!plan.grouped)
    return p.head_dim <= 32   ? launch_attention_rows<DT, 32>(p, t, s)
           : p.head_dim <= 64 ? launch_attention_rows<DT, 64>(p, t, s)
                              : launch_attention_rows<DT, 128>(p, t, s);
  return p.head_dim <= 32   ? launch_attention_cells<DT, 32>(p, t, plan, scratch, s)
         : p.head_dim <= 64 ? launch_attention_cells<DT, 64>(p, t, plan, scratch, s)
                            : launch_attention_cells<DT, 128>(p, t, plan, scratch, s);
}

}  // namespace

BlockAttnPlan attention_blocks_plan(const BlockAttnArgs& p) {
  BlockAttnPlan plan;
  const size_t cells = static_cast<size_t>(p.num_blocks) * p.kv_heads;
  const size_t row_entries = static_cast<size_t>(p.heads) * p.top;  // of a token
  plan.grouped = cells > 0 && cells <= 0x3fffffff && row_entries * p.rows >= 4 * cells;
  if (!plan.grouped) return plan;
  // Entry numbers are 32-bit, and lists of 2^26 entries take half a gigabyte.
  plan.tokens = static_cast<int>(std::min<size_t>(p.rows, std::max<size_t>(1, (size_t{1} << 26) / row_entries)));
  const size_t head_bytes = static_cast<size_t>(plan.tokens) * (p.heads / p.kv_heads) * p.top * (p.head_dim * 4 + 8);
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
