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
#include "common.hpp"
#include "kernels.hpp"

namespace esm_gfx950 {

namespace {

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

// One workgroup per (query, head), its waves taking the row's listed blocks in
// turn, a lane per key for the scores and per dim for the output, with a
// running maximum and sum; the waves' parts meet in LDS. An entry that is
// negative, past the sequence's blocks or a repeat of an earlier one counts for
// nothing; a row without any entry is zero.
template <int DT>
__global__ __launch_bounds__(256) void attention_blocks_kernel(BlockAttnArgs p, SeqTable t) {
  using T = typename ElemOf<DT>::T;
  __shared__ float qs[kMaxHeadDim];
  __shared__ float probs[4][64];
  __shared__ float part_o[4][kMaxHeadDim], part_m[4], part_l[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.x / p.heads, head = blockIdx.x % p.heads;
  const int hk = head / (p.heads / p.kv_heads), dim = p.head_dim;
  const Seq s = seq_at(t, seq_of(t, t.cu_q, 0, row));
  const T* q = static_cast<const T*>(p.q) + static_cast<size_t>(row) * p.ldq + head * dim;
  for (int d = threadIdx.x; d < dim; d += 256) qs[d] = static_cast<float>(q[d]);
  __syncthreads();
  const int* list = p.blocks + (static_cast<size_t>(row) * p.heads + head) * p.top;
  float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (int e = wave; e < p.top; e += 4) {
    const int j = list[e];
    if (j < 0 || j >= s.b1 - s.b0) continue;
    bool repeat = false;
    for (int i = lane; i < e; i += 64) repeat |= list[i] == j;
    if (__ballot(repeat)) continue;
    const int first = s.k0 + j * p.block_size, end = min(first + p.block_size, s.k1);
    for (int c = first; c < end; c += 64) {
      const int n = min(64, end - c);
      float score = -INFINITY;
      if (lane < n) {
        const T* k = static_cast<const T*>(p.k) + static_cast<size_t>(c + lane) * p.ldkv + hk * dim;
        score = 0.0f;
        for (int d = 0; d < dim; ++d) score = __builtin_fmaf(qs[d], static_cast<float>(k[d]), score);
      }
      const float mn = fmaxf(m, wave_max(score));
      const float base = mn == -INFINITY ? 0.0f : mn;
      const float pr = expf(score - base), alpha = expf(m - base);
      l = l * alpha + wave_sum(pr);
      m = mn;
      o0 *= alpha;
      o1 *= alpha;
      probs[wave][lane] = pr;
      __builtin_amdgcn_wave_barrier();
      for (int i = 0; i < n; ++i) {
        const T* v = static_cast<const T*>(p.v) + static_cast<size_t>(c + i) * p.ldkv + hk * dim;
        const float w = probs[wave][i];
        if (lane < dim) o0 = __builtin_fmaf(w, static_cast<float>(v[lane]), o0);
        if (lane + 64 < dim) o1 = __builtin_fmaf(w, static_cast<float>(v[lane + 64]), o1);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  part_o[wave][lane] = o0;
  part_o[wave][lane + 64] = o1;
  if (lane == 0) {
    part_m[wave] = m;
    part_l[wave] = l;
  }
  __syncthreads();
  float mm = -INFINITY;
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, part_m[w]);
  const float base = mm == -INFINITY ? 0.0f : mm;
  float sum = 0.0f;
  for (int w = 0; w < 4; ++w) sum += part_l[w] * expf(part_m[w] - base);
  for (int d = threadIdx.x; d < dim; d += 256) {
    float o = 0.0f;
    for (int w = 0; w < 4; ++w) o += part_o[w][d] * expf(part_m[w] - base);
    static_cast<T*>(p.out)[(static_cast<size_t>(row) * p.heads + head) * dim + d] =
        static_cast<T>(sum == 0.0f ? 0.0f : o / sum);
  }
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

hipError_t launch_attention_blocks(const BlockAttnArgs& p, const SeqTable& t, int type, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(p.rows) * p.heads;
  if (type == kTypeF32)
    attention_blocks_kernel<kTypeF32><<<grid, 256, 0, s>>>(p, t);
  else if (type == kTypeF16)
    attention_blocks_kernel<kTypeF16><<<grid, 256, 0, s>>>(p, t);
  else
    attention_blocks_kernel<kTypeBF16><<<grid, 256, 0, s>>>(p, t);
  return hipGetLastError();
}

}  // namespace esm_gfx950
