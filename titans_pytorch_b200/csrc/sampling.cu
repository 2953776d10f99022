// Token sampling: temperature, repetition penalty, top-k, top-p, min-p and the
// draw itself, from uniform numbers that the caller gives, one row per request.
//
//   z_i = logit_i / T            (fp32; then / penalty for tokens already seen; NaN = -inf)
//   w_i = exp(z_i - max z)
//   top-k:  keep z_i >= the k-th largest z (all ties with it)
//   top-p:  in descending order (ties: lower index first) keep i while the
//           weight in front of it is <= p * sum of the weights left by top-k
//   min-p:  keep w_i >= min_p
//   token:  the first i, by index, whose running sum of kept weights exceeds
//           u * (their sum)
// T <= 0 takes the first largest z.
//
// Weights are held as integers round(w * 2^F), F = 47 for vocabularies up to
// 2^15 and less beyond so that a sum fits 62 bits: integer sums do not depend
// on their order, so a row gives the same token whatever the split, and the
// borders of running sums lie within 2^-47 or so of the real ones (fp32 sums
// would move tokens).
//
// A row is a cluster of 1 to 8 blocks, each with its slice of z in shared
// memory as order-preserving 32-bit keys: the logits are read from memory once.
// Thresholds come from histograms, not from sorting: 1024 bins, first linear in
// z (1/32 wide, from the maximum down), then by key within the chosen bin, until
// a bin decides (one element, or one value).  Two passes settle nearly every
// row.  Each pass ends in one cluster barrier, after which every block sums the
// blocks' bins through distributed shared memory and finds the same answer.
// What bounds it: a single row by that chain of barriers; a large batch of
// large vocabularies by the arithmetic on every element (an fp64 exponential
// and four shared-memory atomics).
#include <cooperative_groups.h>

#include "common.cuh"

namespace tb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kTable = 256;              // entries of the exponential's table
constexpr int kMaxSlice = 40960;         // keys a block can hold
constexpr int kMaxCluster = 8;

// one value for every row, or one per row
struct Setting {
  const float* per_row;
  float all;
  __device__ __forceinline__ float at(int row) const { return per_row ? per_row[row] : all; }
};

struct SampleArgs {
  const void* logits;
  int64_t ls;
  int V, slice, fbits;
  const float* u;
  Setting temp, top_p, min_p, penalty;
  const int64_t* top_k;
  int64_t top_k0;
  const int64_t* seen;  // [B, L] or null
  int64_t seen_s;
  int L;
  int64_t* token;
  float* logprob;
};

// order-preserving map of fp32 to uint32
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kLowest = 0x007fffffu;  // key of -inf

struct Hist {
  uint32_t n[kBins], m0[kBins], m1[kBins], m2[kBins];  // count; weight in 16-bit limbs
};

struct Shared {
  double table[kTable];      // 2^(j / kTable) * 2^F
  Hist hist[2];
  unsigned long long scan[kWarps];
  unsigned long long best;   // this block's largest (key, index)
  unsigned long long mass;   // this block's kept weight
  uint32_t ties;             // this block's elements at the threshold
  uint32_t warp_ties[kWarps];
  unsigned long long warp_mass[kWarps];
  int bin;
  uint32_t bin_n;
  unsigned long long ahead;
  uint32_t edge[2];
};

__device__ __forceinline__ unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, bool RESIDENT>
struct Row {
  const SampleArgs& a;
  Shared& s;
  uint32_t* keys;       // RESIDENT: this block's slice
  uint32_t* seen_bits;  // one bit per element of the slice
  const T* lr;
  float div, pen;
  int row, rank, blocks, i0, n;  // the slice is [i0, i0 + n)
  uint32_t top_key;
  float zmax;
  double zmax_d;
  int level = 0;        // histogram buffers alternate

  __device__ __forceinline__ uint32_t make_key(float logit, int i) const {
    float z = __fdiv_rn(logit, div);
    if (a.seen && (seen_bits[i >> 5] >> (i & 31) & 1u)) z = __fdiv_rn(z, pen);
    return isnan(z) ? kLowest : key_of(z == 0.f ? 0.f : z);
  }
  __device__ __forceinline__ uint32_t key_at(int i) const {
    if constexpr (RESIDENT) return keys[i];
    return make_key(to_f<T>(lr[i0 + i]), i);
  }

  __device__ __forceinline__ void cluster_sync() const {
    if (blocks > 1)
      cg::this_cluster().sync();
    else
      __syncthreads();
  }
  template <typename P> __device__ __forceinline__ const P* peer(const P* p, int r) const {
    return blocks > 1 ? cg::this_cluster().map_shared_rank(p, r) : p;
  }

  // exp(z - zmax) * 2^F, as a double, by the table-driven method (Tang, 1989):
  // x = k ln2 / 256 + r, 2^(k / 256) from the table and the exponent, e^r by its
  // series to r^4 (|r| <= 1.4e-3: 4e-17 beyond it).
  __device__ __forceinline__ double weight(uint32_t key) const {
    if (key == top_key) return s.table[0];
    const double x = (double)value_of(key) - zmax_d;
    if (!(x > -50.0)) return 0.0;  // below 2^-72
    const double t = fma(x, 369.3299304675746, 6755399441055744.0);  // 256 / ln 2; 1.5 * 2^52 rounds to an integer
    const int k = __double2loint(t);
    const double r = fma(t - 6755399441055744.0, -0.0027076061740622863, x);  // ln 2 / 256
    double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double w = p * s.table[k & (kTable - 1)];
    return __hiloint2double(__double2hiint(w) + ((k >> 8) << 20), __double2loint(w));
  }
  // rounded to an integer; w < 2^51
  __device__ __forceinline__ unsigned long long fixed(double w) const {
    return (unsigned long long)(__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffll);
  }

  // bins of the first pass: 1/32 wide below the maximum, the last one open
  __device__ __forceinline__ int linear_bin(uint32_t key) const {
    if (key == top_key) return 0;
    return (int)fminf((zmax - value_of(key)) * 32.f, (float)(kBins - 1));
  }

  // Adds the elements with lo <= key <= hi to this block's histogram.
  template <bool MASS, typename Bin> __device__ __forceinline__ void count(uint32_t lo, uint32_t hi, Bin bin_of) {
    Hist& h = s.hist[level & 1];
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      h.n[i] = 0u;
      if constexpr (MASS) h.m0[i] = h.m1[i] = h.m2[i] = 0u;
    }
    __syncthreads();
    for (int i0_ = 0; i0_ < n; i0_ += kThreads) {
      const int i = i0_ + threadIdx.x;
      const uint32_t key = i < n ? key_at(i) : 0u;
      const bool in = i < n && key >= lo && key <= hi;
      const unsigned active = __ballot_sync(0xffffffffu, in);
      if (!active) continue;
      const int b = in ? bin_of(key) : 0;
      // a warp whose elements share a bin (masked rows, equal logits) adds once
      const int lead = __ffs(active) - 1;
      const int b0 = __shfl_sync(0xffffffffu, b, lead);
      const bool same = __all_sync(0xffffffffu, !in || b == b0);
      unsigned long long m = 0ull;
      if constexpr (MASS)
        if (in) m = fixed(weight(key));
      if (same) {
        if constexpr (MASS) {
          m = warp_sum64(m);  // < 2^52
        }
        if ((threadIdx.x & 31) == lead) {
          atomicAdd(&h.n[b], __popc(active));
          if constexpr (MASS) {
            atomicAdd(&h.m0[b], (uint32_t)(m & 0xffffu));
            atomicAdd(&h.m1[b], (uint32_t)(m >> 16 & 0xffffu));
            atomicAdd(&h.m2[b], (uint32_t)(m >> 32));
          }
        }
      } else if (in) {
        atomicAdd(&h.n[b], 1u);
        if constexpr (MASS) {
          if (m & 0xffffu) atomicAdd(&h.m0[b], (uint32_t)(m & 0xffffu));
          if (m >> 16 & 0xffffu) atomicAdd(&h.m1[b], (uint32_t)(m >> 16 & 0xffffu));
          if (m >> 32) atomicAdd(&h.m2[b], (uint32_t)(m >> 32));
        }
      }
    }
  }

  // Sums the blocks' histograms and finds the bin where the running count (or
  // weight) passes `want`: the first with base + running >= want (count), > want
  // (weight).  Returns the sum over all bins.  `scale_p` >= 0: want becomes
  // floor(scale_p * that sum) first.
  template <bool MASS>
  __device__ __forceinline__ unsigned long long find(unsigned long long base, unsigned long long& want, double scale_p) {
    cluster_sync();
    constexpr int PER = kBins / kThreads;
    const Hist* h = &s.hist[level & 1];
    unsigned long long v[PER];
    uint32_t c[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      v[k] = 0ull;
      c[k] = 0u;
    }
    for (int r = 0; r < blocks; ++r) {
      const Hist* p = peer(h, r);
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int b = threadIdx.x * PER + k;
        c[k] += p->n[b];
        if constexpr (MASS)
          v[k] += (unsigned long long)p->m0[b] + ((unsigned long long)p->m1[b] << 16) +
                  ((unsigned long long)p->m2[b] << 32);
      }
    }
    unsigned long long mine = 0ull;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if constexpr (!MASS) v[k] = c[k];
      mine += v[k];
    }
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    unsigned long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) s.scan[wid] = incl;
    __syncthreads();
    unsigned long long before = 0ull, total = 0ull;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < wid) before += s.scan[w];
      total += s.scan[w];
    }
    if (scale_p >= 0.0) want = (unsigned long long)floor(scale_p * (double)total);
    unsigned long long run = base + before + incl - mine;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const unsigned long long next = run + v[k];
      if (MASS ? (run <= want && next > want) : (run < want && next >= want)) {
        s.bin = threadIdx.x * PER + k;
        s.bin_n = c[k];
        s.ahead = run;
      }
      run = next;
    }
    __syncthreads();
    ++level;
    return total;
  }

  // Key range of a bin of the first pass: its edges by bisection (linear_bin falls as the key grows).
  __device__ __forceinline__ void edges(int bin, uint32_t& lo, uint32_t& hi) {
    if (threadIdx.x < 64 && (threadIdx.x & 31) == 0) {
      const bool upper = threadIdx.x >= 32;
      // lower edge: the smallest key with linear_bin <= bin; upper: the smallest with linear_bin < bin, less one
      uint32_t a_ = kLowest, b_ = top_key;  // linear_bin(top_key) = 0
      const int limit = upper ? bin - 1 : bin;
      if (limit < 0) {
        a_ = top_key + 1u;
      } else {
        while (a_ < b_) {
          const uint32_t mid = a_ + (b_ - a_) / 2;
          if (linear_bin(mid) <= limit) b_ = mid; else a_ = mid + 1;
        }
      }
      s.edge[upper] = upper ? a_ - 1u : a_;
    }
    __syncthreads();
    lo = s.edge[0];
    hi = s.edge[1];
    __syncthreads();
  }

  // The key at which the running count reaches `want`, or the running weight
  // passes it, among keys >= floor_key.  On return every key >= the result is
  // in, except that of `ties_n` keys equal to it only a part may be (weight
  // only; ahead = the weight of larger keys).
  template <bool MASS>
  __device__ __forceinline__ uint32_t select(uint32_t floor_key, unsigned long long want, double scale_p,
                                             unsigned long long& ahead, uint32_t& ties_n, unsigned long long& target) {
    count<MASS>(floor_key, top_key, [&](uint32_t k) { return linear_bin(k); });
    find<MASS>(0ull, want, scale_p);
    target = want;
    uint32_t lo, hi;
    int bin = s.bin;
    uint32_t bn = s.bin_n;
    ahead = s.ahead;
    edges(bin, lo, hi);
    lo = max(lo, floor_key);
    while (true) {
      ties_n = 0;
      // the bin is in as a whole: one element (its weight crosses), or the count ends with it
      if (bn == 1u || (!MASS && ahead + bn == want)) return lo;
      if (lo == hi) {
        ties_n = bn;
        return lo;
      }
      const int sh = max(0, 22 - __clz(hi - lo));  // (hi - lo) >> sh < 1024
      const uint32_t hi0 = hi;
      count<MASS>(lo, hi, [&](uint32_t k) { return (int)((hi0 - k) >> sh); });
      unsigned long long w = want;
      find<MASS>(ahead, w, -1.0);
      bin = s.bin;
      bn = s.bin_n;
      ahead = s.ahead;
      const uint32_t up = hi0 - ((uint32_t)bin << sh);
      lo = max(lo, up - ((1u << sh) - 1u) > up ? 0u : up - ((1u << sh) - 1u));
      hi = up;
    }
  }
};

template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int blocks = (int)cg::this_cluster().num_blocks();
  const int rank = (int)cg::this_cluster().block_rank();
  const int row = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  uint32_t* seen_bits = reinterpret_cast<uint32_t*>(smem + sizeof(Shared));
  uint32_t* keys = seen_bits + (a.seen ? (a.slice + 31) / 32 : 0);
  const float temp = a.temp.at(row);
  const bool greedy = !(temp > 0.f);
  Row<T, RESIDENT> R{a, s, keys, seen_bits, (const T*)a.logits + row * a.ls, greedy ? 1.f : temp,
                     a.penalty.at(row), row, rank, blocks, min(rank * a.slice, a.V), 0, 0u, 0.f, 0.0};
  R.n = min(a.slice, a.V - R.i0);
  for (int j = tid; j < kTable; j += kThreads) s.table[j] = ldexp(exp2((double)j / kTable), a.fbits);
  if (a.seen) {
    for (int i = tid; i < (a.slice + 31) / 32; i += kThreads) seen_bits[i] = 0u;
    __syncthreads();
    for (int i = tid; i < a.L; i += kThreads) {
      const int64_t t = a.seen[row * a.seen_s + i] - R.i0;
      if (t >= 0 && t < R.n) atomicOr(&seen_bits[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
  }
  // keys into shared memory; the largest, and of its ties the first
  uint32_t best = 0u;
  int best_i = 0;
  auto take = [&](float logit, int i) {
    const uint32_t k = R.make_key(logit, i);
    if constexpr (RESIDENT) keys[i] = k;
    if (k > best) {  // a thread's indices grow
      best = k;
      best_i = R.i0 + i;
    }
  };
  constexpr int VEC = Vec16<T>::N;
  const T* src = R.lr + R.i0;
  int done = 0;
  if (((uintptr_t)src & 15) == 0) {
    const int vecs = R.n / VEC;
#pragma unroll 2
    for (int v = tid; v < vecs; v += kThreads) {
      float x[VEC];
      load16<T>(src + v * VEC, x);
#pragma unroll
      for (int k = 0; k < VEC; ++k) take(x[k], v * VEC + k);
    }
    done = vecs * VEC;
  }
  for (int i = done + tid; i < R.n; i += kThreads) take(to_f<T>(src[i]), i);
  unsigned long long packed = R.n > 0 ? ((unsigned long long)best << 32) | (0xffffffffu - (uint32_t)best_i) : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) packed = max(packed, __shfl_xor_sync(0xffffffffu, packed, o));
  if (lane == 0) s.scan[wid] = packed;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) packed = max(packed, s.scan[w]);
    s.best = packed;
  }
  R.cluster_sync();
  for (int r = 0; r < blocks; ++r) packed = max(packed, *R.peer(&s.best, r));
  R.top_key = (uint32_t)(packed >> 32);
  R.zmax = value_of(R.top_key);
  R.zmax_d = (double)R.zmax;
  const int top_i = (int)(0xffffffffu - (uint32_t)packed);
  if (greedy || R.top_key <= kLowest) {
    if (rank == 0 && tid == 0) {
      a.token[row] = top_i;
      a.logprob[row] = greedy ? 0.f : __int_as_float(0x7fffffff);
    }
    R.cluster_sync();  // the peers may still read this block's maximum
    return;
  }
  unsigned long long ahead = 0ull, target = 0ull;
  uint32_t threshold = kLowest, ties_n = 0;
  const int64_t want = a.top_k ? a.top_k[row] : a.top_k0;
  if (want > 0 && want < a.V)
    threshold = R.template select<false>(kLowest, (unsigned long long)want, -1.0, ahead, ties_n, target);
  // how many keys equal to the threshold are in
  unsigned long long ties_in = ~0ull;
  const double p = (double)a.top_p.at(row);
  if (p < 1.0) {
    threshold = R.template select<true>(threshold, 0ull, fmax(p, 0.0), ahead, ties_n, target);
    if (ties_n > 1) {
      const unsigned long long w = R.fixed(R.weight(threshold));
      ties_in = (target - ahead) / w + 1ull;  // w > 0: the running weight crosses within these ties
      if (ties_in >= ties_n) ties_in = ~0ull;
    }
  }
  const double least = (double)a.min_p.at(row) * s.table[0];
  // each warp a contiguous run of the slice, so that running sums follow the index
  const int per = ((R.n + kWarps - 1) / kWarps + 31) & ~31;
  const int w0 = min(wid * per, R.n), w1 = min(w0 + per, R.n);
  unsigned long long tie_base = 0ull;
  if (ties_in != ~0ull) {  // the same in every block of the row
    uint32_t t = 0;
    for (int i = w0; i < w1; i += 32) t += __popc(__ballot_sync(0xffffffffu, i + lane < w1 && R.key_at(i + lane) == threshold));
    if (lane == 0) s.warp_ties[wid] = t;
    __syncthreads();
    if (tid == 0) {
      uint32_t all = 0;
      for (int w = 0; w < kWarps; ++w) all += s.warp_ties[w];
      s.ties = all;
    }
    R.cluster_sync();
    for (int r = 0; r < rank; ++r) tie_base += *R.peer(&s.ties, r);
    for (int w = 0; w < wid; ++w) tie_base += s.warp_ties[w];
  }
  // kept weight of element i + lane; `tie` counts the threshold's ties in front of this step
  auto kept = [&](int i, unsigned long long& tie) -> unsigned long long {
    const uint32_t key = i + lane < w1 ? R.key_at(i + lane) : 0u;
    bool in = key >= threshold && i + lane < w1;
    if (ties_in != ~0ull) {
      const unsigned eq = __ballot_sync(0xffffffffu, in && key == threshold);
      if (key == threshold && tie + __popc(eq & ((1u << lane) - 1u)) >= ties_in) in = false;
      tie += __popc(eq);
    }
    if (!in) return 0ull;
    const double w = R.weight(key);
    return w >= least ? R.fixed(w) : 0ull;
  };
  unsigned long long mine = 0ull, tie = tie_base;
  for (int i = w0; i < w1; i += 32) mine += kept(i, tie);
  mine = warp_sum64(mine);
  if (lane == 0) s.warp_mass[wid] = mine;
  __syncthreads();
  if (tid == 0) {
    unsigned long long all = 0ull;
    for (int w = 0; w < kWarps; ++w) all += s.warp_mass[w];
    s.mass = all;
  }
  R.cluster_sync();
  unsigned long long total = 0ull, base = 0ull;
  for (int r = 0; r < blocks; ++r) {
    const unsigned long long m = *R.peer(&s.mass, r);
    if (r < rank) base += m;
    total += m;
  }
  for (int w = 0; w < wid; ++w) base += s.warp_mass[w];
  // run > u * total for the integer run means run > floor(u * total); u = 1 ends at the last kept token
  unsigned long long goal = (unsigned long long)floor(fmax((double)a.u[row], 0.0) * (double)total);
  goal = min(goal, total - 1ull);
  if (base <= goal && goal < base + mine) {  // one warp of the row
    tie = tie_base;
    for (int i = w0; i < w1; i += 32) {
      const unsigned long long m = kept(i, tie);
      unsigned long long incl = m;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      const unsigned over = __ballot_sync(0xffffffffu, base + incl > goal);
      if (over) {
        if (lane == __ffs(over) - 1) {
          a.token[row] = R.i0 + i + lane;
          const float z = value_of(R.key_at(i + lane));
          const double x = R.key_at(i + lane) == R.top_key ? 0.0 : (double)z - R.zmax_d;
          a.logprob[row] = (float)(x - log((double)total / s.table[0]));
        }
        break;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  R.cluster_sync();  // the peers may still read this block's sums
}

template <typename T, bool RESIDENT>
void launch_sample(const SampleArgs& a, int64_t B, int cluster, size_t smem) {
  static bool set[64] = {};
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(sample_kernel<T, RESIDENT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)(sizeof(Shared) + kMaxSlice * 4 + kMaxSlice / 8)));
    if (dev < 64) set[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(B * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, sample_kernel<T, RESIDENT>, a));
}

}  // namespace

std::vector<at::Tensor> sample_tokens(const at::Tensor& logits, const at::Tensor& u,
                                      const c10::optional<at::Tensor>& temp, double temp0,
                                      const c10::optional<at::Tensor>& top_k, int64_t top_k0,
                                      const c10::optional<at::Tensor>& top_p, double top_p0,
                                      const c10::optional<at::Tensor>& min_p, double min_p0,
                                      const c10::optional<at::Tensor>& penalty, double penalty0,
                                      const c10::optional<at::Tensor>& seen) {
  const char* what = "sample_tokens";
  TB_CHECK_CUDA(logits);
  TORCH_CHECK(logits.dim() == 2 && logits.stride(1) == 1, what, ": logits must be [B, V] with contiguous rows");
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V >= 1 && V <= (1 << 19), what, ": a vocabulary of 1 to 2^19 tokens");
  auto check_rows = [&](const at::Tensor& t, at::ScalarType type, const char* name) {
    TORCH_CHECK(t.device() == logits.device() && t.scalar_type() == type && t.dim() == 1 && t.size(0) == B &&
                    t.is_contiguous(),
                what, ": ", name, " must be a contiguous ", type, " [", B, "] on the logits' device");
  };
  check_rows(u, at::kFloat, "uniform");
  auto setting = [&](const c10::optional<at::Tensor>& t, double all, const char* name) {
    Setting s{nullptr, (float)all};
    if (t.has_value() && t->defined()) {
      check_rows(*t, at::kFloat, name);
      s.per_row = t->data_ptr<float>();
    }
    return s;
  };
  const at::cuda::CUDAGuard g(logits.device());
  at::Tensor token = at::empty({B}, logits.options().dtype(at::kLong));
  at::Tensor logprob = at::empty({B}, logits.options().dtype(at::kFloat));
  if (B == 0) return {token, logprob};
  SampleArgs a{};
  a.logits = logits.data_ptr();
  a.ls = logits.stride(0);
  a.V = (int)V;
  a.u = u.data_ptr<float>();
  a.temp = setting(temp, temp0, "temperature");
  a.top_p = setting(top_p, top_p0, "top_p");
  a.min_p = setting(min_p, min_p0, "min_p");
  a.penalty = setting(penalty, penalty0, "repetition_penalty");
  a.top_k0 = top_k0;
  if (top_k.has_value() && top_k->defined()) {
    check_rows(*top_k, at::kLong, "top_k");
    a.top_k = top_k->data_ptr<int64_t>();
  }
  a.token = token.data_ptr<int64_t>();
  a.logprob = logprob.data_ptr<float>();
  if (seen.has_value() && seen->defined() && seen->size(1) > 0) {
    TORCH_CHECK(seen->device() == logits.device() && seen->scalar_type() == at::kLong && seen->dim() == 2 &&
                    seen->size(0) == B && seen->stride(1) == 1 && seen->size(1) < (1ll << 31),
                what, ": generated must be int64 [", B, ", n] with contiguous rows on the logits' device");
    a.seen = seen->data_ptr<int64_t>();
    a.seen_s = seen->stride(0);
    a.L = (int)seen->size(1);
  }
  // as many blocks a row as the GPU holds at once (two an SM), at least enough for the row to fit their memory
  int cluster = 1;
  while (cluster < kMaxCluster && (B * cluster * 2 <= 2 * num_sms() || (V + cluster - 1) / cluster > kMaxSlice) &&
         V / (cluster * 2) >= 512)
    cluster *= 2;
  a.slice = (int)(((V + cluster - 1) / cluster + 31) / 32 * 32);
  TORCH_CHECK(B * cluster < (1ll << 31), what, ": too many rows in one call");
  int bits = 15;
  while ((1ll << bits) < V) ++bits;
  a.fbits = 62 - bits;
  const bool resident = a.slice <= kMaxSlice;
  const size_t smem = sizeof(Shared) + (a.seen ? (a.slice + 31) / 32 * 4 : 0) + (resident ? (size_t)a.slice * 4 : 0);
  TB_DISPATCH_FLOAT(logits.scalar_type(), what, [&] {
    if (resident)
      launch_sample<scalar_t, true>(a, B, cluster, smem);
    else
      launch_sample<scalar_t, false>(a, B, cluster, smem);
  });
  check_launch(what);
  return {token, logprob};
}

}  // namespace tb
