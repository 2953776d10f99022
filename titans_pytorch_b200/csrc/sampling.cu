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
// Weights are held as integers round(w * 2^F): integer sums are exact and do not
// depend on their order, so the same row always gives the same token.  F = 47,
// 46, 44, 41, 38 for vocabularies up to 2^15, 2^16, 2^17, 2^18, 2^19, so that sums
// of V of them fit.  A weight below half a unit counts nothing (it cannot be
// drawn, not even by u = 0), and a running sum is off by V half units at most,
// as where a tail of V equal weights is rounded away: by 2^-33, 2^-31, 2^-28,
// 2^-24, 2^-20 of the largest weight.
//
// Nothing is sorted; a row is passed over two to four times (from L2 after the
// first), or up to 13 times by one block where a border lies among more
// elements than the list holds (up to four passes narrow the count, one sums what
// it left, up to four narrow the weight, one looks for ties):
//   1. the maximum (greedy rows: and its index; they are done);
//   2. counts in 1024 bins linear in z, 1/32 wide below the maximum, and for
//      top-p the exact sum of all weights;
//   3. from the counts follow the bin of the k-th largest, or, as a bin's
//      elements weigh the same within 3 %, two bins between which top-p's border
//      must lie: their elements go to a list in shared memory, which is narrowed
//      by histograms over the keys (order-preserving 32-bit images of z) until a
//      bin decides: one element, or one value.  If they do not fit, the row is
//      passed over instead;
//   4. the draw is the same search over the index: kept weight in 1024 index
//      bins, then the elements of one bin.
// Rows without a filter need 1 and 4 only.  Where min-p cuts above top-p's
// border for certain, which the counts tell, top-p is left out.  After 3 the draw
// works on the list if that holds everything that may be kept.
//
// One block does all of this for a row; while SMs are free, up to seven more
// take parts of the passes and add their counts, sums and list entries to its
// shared memory.  (Letting every block of a cluster sum all blocks' bins itself
// cost 2.5 us a search, and keeping the row in shared memory gained nothing.)
// What bounds it: one row, the chain of barriers (a cluster's costs about 1 us
// with the read behind it); many rows, the instructions of the passes: 148 rows of
// 131072 fp32 logits with top-p and min-p execute 94 an element, every SM issuing
// in 61 % of its cycles, and one block an SM leaves a row's barriers uncovered.
#include <cooperative_groups.h>

#include "common.cuh"

namespace tb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kBins = kThreads;          // one a thread
constexpr int kTable = 16;               // entries of the exponential's table
constexpr int kShort = kThreads / 8;     // a list that is compared all against all
constexpr int kSharedLimit = 226 * 1024;

// one value for every row, or one per row
struct Setting {
  const float* per_row;
  float all;
  __device__ __forceinline__ float at(int row) const { return per_row ? per_row[row] : all; }
};

struct SampleArgs {
  const void* logits;
  int64_t ls;
  int V, slice, fbits, limb, list_cap, index_shift;
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

using u64 = unsigned long long;

// order-preserving map of fp32 to uint32
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kLowest = 0x007fffffu;  // key of -inf

struct __align__(16) Shared {
  double table[kTable];  // 2^(j / kTable) * 2^F
  uint32_t n[kBins], m0[kBins], m1[kBins], m2[kBins];  // count; weight in three limbs (shared memory adds 32 bits)
  u64 scan[kWarps];
  double scan_d[kWarps][2];
  int bin, bin_lo, bin_hi, at;
  uint32_t bin_n;
  u64 ahead;
  uint32_t edge[2];
  // of the row's first block: what the others add to, and what it tells them
  u64 best[8], total[8];  // by block (64-bit atomics on the first block's were tried and gave wrong maxima; cause not found)
  uint32_t lo, hi, threshold;
  int list_n, route, tie_last;
};

// what the first block makes the others do after the counts
enum Route : int { DRAW = 0, LIST_ALL = 1, LIST_BORDER = 2, ALONE = 3 };

template <typename V> __device__ __forceinline__ V warp_scan(V v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

template <typename T>
struct Row {
  static constexpr int VEC = 8 / sizeof(T);
  const SampleArgs& a;
  Shared& s;
  const uint32_t* seen_bits;
  uint2* list;        // (key, index)
  const T* lr;
  float div, pen;
  bool vec;           // 8-byte loads
  bool plain;         // z is the logit
  bool penalised;
  bool listed = false;
  float zmax_f = 0.f, bin_top = 0.f;
  uint32_t top_key = 0u;
  double zmax = 0.0;

  __device__ __forceinline__ void set_top(uint32_t key) {
    top_key = key;
    zmax_f = value_of(key);
    bin_top = fminf(zmax_f, 3.4028234e38f);  // an infinite maximum is in bin 0 too
    zmax = (double)zmax_f;
  }
  static __device__ __forceinline__ void cluster_sync(int blocks) {
    if (blocks > 1)
      cg::this_cluster().sync();
    else
      __syncthreads();
  }

  // z of an element: -0 becomes 0; NaN stays NaN (its key is that of -inf)
  __device__ __forceinline__ float scaled(float logit, int i) const {
    float z = div == 1.f ? logit : __fdiv_rn(logit, div);
    if (penalised && (seen_bits[i >> 5] >> (i & 31) & 1u)) z = __fdiv_rn(z, pen);
    return z + 0.f;
  }
  static __device__ __forceinline__ uint32_t key_or_low(float z) { return isnan(z) ? kLowest : key_of(z); }
  __device__ __forceinline__ uint32_t key_at(int i) const { return key_or_low(scaled(to_f<T>(lr[i]), i)); }

  // f(z[VEC], index of the first, how many) for groups of elements of [i0, i1);
  // the lanes of a warp call it together (none behind the end).
  template <typename F> __device__ __forceinline__ void groups(int i0, int i1, F f) const {
    if (plain)
      groups_of<false>(i0, i1, f);
    else
      groups_of<true>(i0, i1, f);
  }
  template <bool SCALE, typename F> __device__ __forceinline__ void groups_of(int i0, int i1, F f) const {
    // Two vectors in flight a thread, each register reloaded as soon as it is
    // used (moving them along would wait for the loads).  Whole blocks of
    // vectors first, so that the loop over them checks nothing.
    constexpr int AHEAD = 2;
    int rest = i0;
    if (vec) {
      const int v0 = i0 / VEC + threadIdx.x;  // i0 is a multiple of VEC
      const int full = (i1 / VEC - i0 / VEC) / kThreads;
      const uint2* src = reinterpret_cast<const uint2*>(lr) + v0;
      uint2 x[AHEAD];
#pragma unroll
      for (int q = 0; q < AHEAD; ++q)
        if (q < full) x[q] = src[q * kThreads];
#pragma unroll 1
      for (int b = 0; b < full; b += AHEAD) {
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
          if (b + q >= full) break;
          union { uint2 raw; T e[VEC]; } cur;
          cur.raw = x[q];
          if (b + q + AHEAD < full) x[q] = src[(b + q + AHEAD) * kThreads];
          const int i = (v0 + (b + q) * kThreads) * VEC;
          float z[VEC];
#pragma unroll
          for (int k = 0; k < VEC; ++k) z[k] = SCALE ? scaled(to_f<T>(cur.e[k]), i + k) : to_f<T>(cur.e[k]) + 0.f;
          f(z, i, VEC);
        }
      }
      rest = i0 + full * kThreads * VEC;
    }
    // the rest, and rows that are not aligned
#pragma unroll 1
    for (int b = rest; b < i1; b += kThreads * VEC) {
      float z[VEC];
      const int i = b + threadIdx.x * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        z[k] = i + k < i1 ? (SCALE ? scaled(to_f<T>(lr[i + k]), i + k) : to_f<T>(lr[i + k]) + 0.f) : 0.f;
      f(z, i, max(0, min(VEC, i1 - i)));
    }
  }
  // f(key, index) for every element of the list, or of the row; the lanes of a warp call it together (key 0: none).
  template <typename F> __device__ __forceinline__ void each(F f) const {
    if (listed) {
      const int n = s.list_n;
#pragma unroll 1
      for (int b = 0; b < n; b += kThreads) {
        const int i = b + threadIdx.x;
        const uint2 e = i < n ? list[i] : make_uint2(0u, 0u);
        f(e.x, (int)e.y);
      }
    } else {
      groups(0, a.V, [&](const float (&z)[VEC], int i, int n) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) f(k < n ? key_or_low(z[k]) : 0u, i + k);
      });
    }
  }

  // exp(z - zmax) * 2^F, as a double, by the table-driven method (Tang, 1989):
  // x = k ln2 / 16 + r, 2^(k / 16) from the table and the exponent, e^r by its
  // series to r^6 (|r| <= 0.022: 5e-16 beyond it).  Sixteen doubles fill the
  // shared-memory banks once, so lanes never wait for one another.
  // Without branches, so that the chains of a vector's elements overlap.
  __device__ __forceinline__ double weight(uint32_t key) const {
    // the fp32 value as a double by its bits (a conversion takes eight times an
    // fp64 operation): zero and denormals come out below 2^-126, infinity as
    // 2^128, which is all the same to the difference
    const uint32_t b = __float_as_uint(value_of(key));
    const double v = __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(b << 29));
    return weight_at(key == top_key ? 0.0 : v - zmax);
  }
  __device__ __forceinline__ double weight_at(double x) const {
    x = x > -60.0 ? x : -60.0;  // 2^-86: 0 once rounded
    const double t = fma(x, 23.083120654223414, 6755399441055744.0);  // 16 / ln 2; 1.5 * 2^52 rounds to an integer
    const int k = __double2loint(t);
    const double r = fma(t - 6755399441055744.0, -0.04332169878499658, x);  // ln 2 / 16
    double p = fma(r, 1.0 / 720.0, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double w = p * s.table[k & (kTable - 1)];
    return __hiloint2double(__double2hiint(w) + ((k >> 4) << 20), __double2loint(w));
  }
  // rounded to an integer; w < 2^51
  __device__ __forceinline__ u64 fixed(double w) const {
    return (u64)(__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffll);
  }

  // bins of the counts: bin b is within 1/64 of zmax - b / 32; the last (with NaN) is open
  __device__ __forceinline__ int linear_bin(float z) const {
    const float b = fmaxf(fminf((bin_top - z) * 32.f, (float)(kBins - 1)), 0.f);
    return __float_as_int(b + 8388608.f) & (kBins - 1);  // 2^23 rounds to an integer
  }

  template <bool MASS> __device__ __forceinline__ void clear() {
    s.n[threadIdx.x] = 0u;
    if constexpr (MASS) s.m0[threadIdx.x] = s.m1[threadIdx.x] = s.m2[threadIdx.x] = 0u;
    __syncthreads();
  }
  __device__ __forceinline__ void add_mass(int b, u64 m) {
    const uint32_t mask = (1u << a.limb) - 1u;
    atomicAdd(&s.m0[b], (uint32_t)m & mask);
    atomicAdd(&s.m1[b], (uint32_t)(m >> a.limb) & mask);
    atomicAdd(&s.m2[b], (uint32_t)(m >> 2 * a.limb));
  }
  __device__ __forceinline__ u64 bin_mass(int b) const {
    return (u64)s.m0[b] + ((u64)s.m1[b] << a.limb) + ((u64)s.m2[b] << 2 * a.limb);
  }
  // Adds each lane's weight of its elements, whose indices follow the lane's, to
  // their index bin; the lanes of a bin (a power of two) add up first.
  __device__ __forceinline__ void add_by_index(int i, u64 m) {
    const int lanes = min((1 << a.index_shift) / VEC, 32);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      if (o >= lanes) break;
      m += __shfl_xor_sync(0xffffffffu, m, o);
    }
    if (m && (threadIdx.x & (lanes - 1)) == 0) add_mass(i >> a.index_shift, m);
  }
  // Adds the elements `in` to bins b; a warp whose elements share a bin (equal logits) adds once.
  __device__ __forceinline__ void add(bool in, int b, u64 m) {
    const unsigned active = __ballot_sync(0xffffffffu, in);
    if (!active) return;
    const int lead = __ffs(active) - 1;
    const int lead_b = __shfl_sync(0xffffffffu, b, lead);  // by every lane, so not inside the ||
    const bool same = __all_sync(0xffffffffu, !in || b == lead_b);
    if (in) atomicAdd(&s.n[b], 1u);
    if (same) {
      if (!in) m = 0ull;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);  // < 2^52
    }
    if (same ? (threadIdx.x & 31) == lead : in) add_mass(b, m);
  }

  __device__ __forceinline__ u64 block_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) s.scan[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s.scan[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    return v;
  }
  // sum of the threads in front, and of all
  __device__ __forceinline__ u64 block_before(u64 v, u64& all) {
    const u64 incl = warp_scan(v);
    if ((threadIdx.x & 31) == 31) s.scan[threadIdx.x >> 5] = incl;
    __syncthreads();
    const u64 w = warp_scan(s.scan[threadIdx.x & 31]);
    const int wid = threadIdx.x >> 5;
    const u64 before = __shfl_sync(0xffffffffu, w, max(wid - 1, 0));
    all = __shfl_sync(0xffffffffu, w, 31);
    __syncthreads();
    return (wid ? before : 0ull) + incl - v;
  }

  // The bin where base + the running count (MASS: weight) reaches (passes) `want`: s.bin, s.bin_n, s.ahead.
  template <bool MASS> __device__ __forceinline__ void find(u64 base, u64 want) {
    __syncthreads();
    const int b = threadIdx.x;
    const uint32_t c = s.n[b];
    const u64 v = MASS ? bin_mass(b) : (u64)c;
    u64 all;
    const u64 run = base + block_before(v, all), next = run + v;
    if (MASS ? (run <= want && next > want) : (run < want && next >= want)) {
      s.bin = b;
      s.bin_n = c;
      s.ahead = run;
    }
    __syncthreads();
  }

  // From the counts: the bins between which the running weight passes `want`
  // (s.bin_lo, s.bin_hi).  The elements of bin b weigh between
  // exp(-(b + 1/2) / 32) and exp(-(b - 1/2) / 32), with 1e-5 for the rounding of
  // z - zmax and 1 for that of a weight.  `want` < 0: p times the least that all
  // weigh; then s.bin tells whether bins 0 .. last weigh no more than that for certain.
  __device__ __forceinline__ void bracket(double want, double p, int last) {
    __syncthreads();
    const int b = threadIdx.x;
    const uint32_t c = s.n[b];
    const double up = c * (fmin(weight_at((0.5 - b) * (1.0 / 32.0)) * (1.0 + 1e-5), s.table[0]) + 1.0);
    const double low = b == kBins - 1 ? 0.0 : c * fmax(weight_at((-0.5 - b) * (1.0 / 32.0)) * (1.0 - 1e-5) - 1.0, 0.0);
    if (b == 0) {
      s.bin_lo = kBins - 1;
      s.bin_hi = s.bin = 0;
    }
    const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const double iu = warp_scan(up), il = warp_scan(low);
    if (lane == 31) {
      s.scan_d[wid][0] = iu;
      s.scan_d[wid][1] = il;
    }
    __syncthreads();
    const double su = warp_scan(s.scan_d[lane][0]), sl = warp_scan(s.scan_d[lane][1]);
    const double all_l = __shfl_sync(0xffffffffu, sl, 31);
    const double bu = __shfl_sync(0xffffffffu, su, max(wid - 1, 0)), bl = __shfl_sync(0xffffffffu, sl, max(wid - 1, 0));
    const double ru = (wid ? bu : 0.0) + iu, rl = (wid ? bl : 0.0) + il - low;
    if (want < 0.0) {
      if (b == last) s.bin = ru * (1.0 + 1e-9) + 1.0 < p * all_l;
    } else {
      if (c && ru > want * (1.0 - 1e-12) - 1.0) atomicMin(&s.bin_lo, b);
      if (c && rl <= want * (1.0 + 1e-12)) atomicMax(&s.bin_hi, b);
    }
    __syncthreads();
  }

  // Key range of bins b0 .. b1 of the counts (linear_bin falls as the key
  // grows): warp 0 finds the smallest key with linear_bin <= b1, warp 1 the
  // smallest with linear_bin < b0, each in seven 32-way steps.
  __device__ __forceinline__ void edges(int b0, int b1, uint32_t& lo, uint32_t& hi) {
    const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (wid < 2) {
      const int limit = wid ? b0 - 1 : b1;
      uint32_t at;  // the smallest key with linear_bin <= limit, or top_key + 1
      uint32_t a_ = kLowest, b_ = top_key + 1u;  // the answer lies in [a_, b_]
      while (a_ < b_) {
        const uint32_t step = ((b_ - a_) >> 5) + 1u;
        const uint32_t probe = step * lane < b_ - a_ ? a_ + step * lane : b_;
        const unsigned yes = __ballot_sync(0xffffffffu, probe >= b_ || linear_bin(value_of(probe)) <= limit);
        // (the probe at b_ counts as found, so some lane has one unless all probes lie beneath it)
        const int first = yes ? __ffs(yes) - 1 : 32;
        const uint32_t found = __shfl_sync(0xffffffffu, probe, first & 31);
        if (first == 0) {
          b_ = a_;
        } else {
          if (first < 32) b_ = found;
          a_ = min(a_ + step * (first - 1) + 1u, b_);
        }
      }
      at = a_;
      if (lane == 0) s.edge[wid] = wid ? at - 1u : at;
    }
    __syncthreads();
    lo = s.edge[0];
    hi = s.edge[1];
    __syncthreads();
  }

  // Narrows [lo, hi] to the key at which the running count (MASS: weight) in
  // front of which `ahead` lies reaches (passes) `want`.  Keys >= the result are
  // in; MASS with ties_n > 1: of the ties_n keys equal to it only a part may be,
  // `ahead` being the weight of larger keys.  `first`: ahead is not known yet.
  template <bool MASS>
  __device__ __forceinline__ uint32_t narrow(uint32_t lo, uint32_t hi, u64 want, u64& ahead, uint32_t& ties_n,
                                             bool first) {
    ties_n = 0;
    while (true) {
      const int sh = max(0, 22 - __clz(hi - lo));  // (hi - lo) >> sh < 1024
      clear<MASS>();
      u64 sum = 0ull;
      each([&](uint32_t key, int) {
        const bool in = key >= lo && key <= hi;
        const int b = in ? (int)((hi - key) >> sh) : 0;
        if constexpr (MASS) {
          if (first && key > hi) sum += fixed(weight(key));
          add(in, b, in ? fixed(weight(key)) : 0ull);
        } else {
          if (in) atomicAdd(&s.n[b], 1u);
        }
      });
      if (MASS && first) ahead = block_sum(sum);
      first = false;
      find<MASS>(ahead, want);
      const uint32_t bn = s.bin_n, up = hi - ((uint32_t)s.bin << sh);
      ahead = s.ahead;
      const uint32_t width = (1u << sh) - 1u;
      lo = up - lo > width ? up - width : lo;
      hi = up;
      // the bin is in as a whole: one element (its weight crosses), or the count ends with it
      if (bn == 1u || (!MASS && ahead + bn == want)) return lo;
      if (lo == hi) {
        ties_n = bn;
        return lo;
      }
      __syncthreads();  // s.bin is read before the next search writes it
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  constexpr int VEC = Row<T>::VEC;
  const cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  Shared& first = *cluster.map_shared_rank(&s, 0);
  uint32_t* seen_bits = reinterpret_cast<uint32_t*>(smem + sizeof(Shared));
  const int seen_words = a.seen ? ((a.V + 31) / 32 + 3) / 4 * 4 : 0;
  uint2* list = reinterpret_cast<uint2*>(seen_bits + seen_words);
  uint2* first_list = cluster.map_shared_rank(list, 0);
  // all settings at once: each is a memory latency of its own
  const float temp = a.temp.at(row), pen = a.penalty.at(row), min_p = fminf(fmaxf(a.min_p.at(row), 0.f), 1.f);  // NaN: 0
  const double p = (double)a.top_p.at(row), u = (double)a.u[row];
  const int64_t want_k = a.top_k ? a.top_k[row] : a.top_k0;
  const bool greedy = !(temp > 0.f);
  const T* lr = (const T*)a.logits + row * a.ls;
  Row<T> R{a, s, seen_bits, list, lr, greedy ? 1.f : temp, pen, ((uintptr_t)lr & 7) == 0,
           (greedy || temp == 1.f) && (a.seen == nullptr || pen == 1.f), a.seen != nullptr && pen != 1.f};
  if (blocks > 1) asm volatile("barrier.cluster.arrive.aligned;\n" ::: "memory");
  if (tid < kTable) s.table[tid] = ldexp(exp2((double)tid / kTable), a.fbits);
  s.n[tid] = s.m0[tid] = s.m1[tid] = s.m2[tid] = 0u;
  if (tid == 0) s.list_n = s.bin = 0;
  if (R.penalised) {
    for (int i = tid; i < seen_words; i += kThreads) seen_bits[i] = 0u;
    __syncthreads();
    for (int i = tid; i < a.L; i += kThreads) {
      const int64_t t = a.seen[row * a.seen_s + i];
      if (t >= 0 && t < a.V) atomicOr(&seen_bits[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
  }
  // 1. the largest of this block's part, and of the row
  const int i0 = min(rank * a.slice, a.V), i1 = min(i0 + a.slice, a.V);
  u64 packed = 0ull;
  if (greedy) {  // of its ties the first
    R.groups(i0, i1, [&](const float (&z)[VEC], int i, int n) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (k < n) packed = max(packed, ((u64)R.key_or_low(z[k]) << 32) | (0xffffffffu - (uint32_t)(i + k)));
    });
  } else {
    float zm = -INFINITY;
    R.groups(i0, i1, [&](const float (&z)[VEC], int, int n) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (k < n) zm = fmaxf(zm, z[k]);
    });
    packed = (u64)key_of(zm) << 32;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) packed = max(packed, __shfl_xor_sync(0xffffffffu, packed, o));
  if (lane == 0) s.scan[wid] = packed;
  __syncthreads();
  // a block's shared memory may be written once it runs
  if (blocks > 1) asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
  if (wid == 0) {
    packed = s.scan[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) packed = max(packed, __shfl_xor_sync(0xffffffffu, packed, o));
    if (lane < blocks) cluster.map_shared_rank(&s, lane)->best[rank] = packed;  // to every block
  }
  R.cluster_sync(blocks);
  packed = s.best[0];
  for (int r = 1; r < blocks; ++r) packed = max(packed, s.best[r]);
  R.set_top((uint32_t)(packed >> 32));
  if (greedy || R.top_key <= kLowest) {  // alike in every block
    if (rank == 0 && tid == 0) {
      a.token[row] = greedy ? (int64_t)(0xffffffffu - (uint32_t)packed) : 0;
      a.logprob[row] = greedy ? 0.f : __int_as_float(0x7fffffff);
    }
    return;
  }
  const bool by_count = want_k > 0 && want_k < a.V;
  bool by_mass = p < 1.0;
  // below this key exp(z - zmax) < min_p for certain, with room for the logarithm's rounding and that of the sum
  uint32_t min_cut = kLowest;
  if (min_p > 0.f)
    min_cut = max(min(key_of(R.zmax_f + (logf(min_p) - 1e-3f) - fabsf(R.zmax_f) * 1e-6f), R.top_key), kLowest);
  const int ish = a.index_shift;
  const double least = (double)min_p * s.table[0];
  uint32_t lo = kLowest, hi = R.top_key, threshold = kLowest, ties_n = 0;
  u64 ahead = 0ull, want = 0ull, total = 0ull;
  u64 ties_in = ~0ull;  // how many keys equal to the threshold are in
  int tie_last = a.V, route = DRAW;
  const bool filtered = by_count || by_mass || min_p > 0.f;
  if (filtered) {
    // 2. counts; the sum of all weights where top-p alone decides
    const bool sum_now = by_mass && !by_count && !(min_p > 0.f);
    u64 sum = 0ull;
    R.groups(i0, i1, [&](const float (&z)[VEC], int, int n) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (k < n) atomicAdd(&s.n[R.linear_bin(z[k])], 1u);
      if (sum_now)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const u64 w = R.fixed(R.weight(R.key_or_low(z[k])));
          sum += k < n ? w : 0ull;
        }
    });
    if (sum_now) {
      sum = R.block_sum(sum);
      if (tid == 0) first.total[rank] = sum;
    } else {
      __syncthreads();
    }
    if (rank > 0 && s.n[tid]) atomicAdd(&first.n[tid], s.n[tid]);
    R.cluster_sync(blocks);
    // where min-p cuts above top-p's border for certain, top-p decides nothing
    if (by_mass && !by_count && min_p > 0.f) {
      if (rank == 0) {
        R.bracket(-1.0, fmax(p, 0.0), R.linear_bin(value_of(min_cut)));
        if (tid == 0) s.route = s.bin;
      }
      R.cluster_sync(blocks);
      by_mass = first.route == 0;
      if (by_mass) {
        u64 m = 0ull;
        R.groups(i0, i1, [&](const float (&z)[VEC], int, int n) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            const u64 w = R.fixed(R.weight(R.key_or_low(z[k])));
            m += k < n ? w : 0ull;
          }
        });
        m = R.block_sum(m);
        if (tid == 0) first.total[rank] = m;
      }
      R.cluster_sync(blocks);
    }
  }
  if (filtered) {
    bool open = false;  // the k-th largest lies strictly inside [lo, hi]
    if (rank == 0) {
      if (by_count) {
        want = (u64)want_k;
        R.template find<false>(0ull, want);
        ahead = s.ahead;
        open = !(s.bin_n == 1u || ahead + s.bin_n == want);
        R.edges(s.bin, s.bin, lo, hi);
      } else if (!by_mass) {  // min-p alone
        lo = min_cut;
      } else {
        for (int r = 0; r < blocks; ++r) total += s.total[r];
        want = (u64)floor(fmax(p, 0.0) * (double)total);
        R.bracket((double)want, 0.0, 0);
        R.edges(s.bin_lo, max(s.bin_lo, s.bin_hi), lo, hi);
      }
      const int last = R.linear_bin(value_of(lo)), past = R.linear_bin(value_of(hi));
      const u64 all = R.block_sum(tid <= last ? s.n[tid] : 0u);
      const u64 border = R.block_sum(tid <= last && tid >= past ? s.n[tid] : 0u);
      // A long list is drawn from by one block, the row by all.  131072 fp32 logits, as a row / as a list: one row with
      // 11000 to 21000 candidates 22 / 26 us; but 256 rows, a block each, with 5000 candidates 210 / 136 us.
      const u64 most = by_count ? (u64)a.list_cap : min((u64)a.list_cap, (u64)(4 * kThreads));
      route = all <= most                                            ? LIST_ALL
              : !by_count && !by_mass                                ? DRAW
              : !by_count && border <= (u64)a.list_cap ? LIST_BORDER : ALONE;
      if (tid == 0) {
        s.lo = lo;
        s.hi = hi;
        s.route = route;
      }
    }
    R.cluster_sync(blocks);
    if (rank > 0) {
      lo = first.lo;
      hi = first.hi;
      route = first.route;
    }
    // 3. the list, and the weight in front of it
    if (route == LIST_ALL || route == LIST_BORDER) {
      const float lo_z = value_of(lo), hi_z = route == LIST_ALL ? INFINITY : value_of(hi);
      const float sum_z = by_mass && !by_count ? value_of(hi) : INFINITY;
      const bool all_in = lo <= kLowest;
      u64 m = 0ull;
      R.groups(i0, i1, [&](const float (&z)[VEC], int i, int n) {
        bool over = false;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          if (k < n && ((z[k] >= lo_z && z[k] <= hi_z) || (all_in && !(z[k] > hi_z))))  // few elements are
            first_list[atomicAdd(&first.list_n, 1)] = make_uint2(R.key_or_low(z[k]), (uint32_t)(i + k));
          over |= k < n && z[k] > sum_z;
        }
        if (__any_sync(0xffffffffu, over))
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            const u64 w = R.fixed(R.weight(key_of(z[k])));
            m += k < n && z[k] > sum_z ? w : 0ull;
          }
      });
      m = R.block_sum(m);
      if (tid == 0) first.total[rank] = m;
    }
    R.cluster_sync(blocks);
    if (rank > 0 && route == LIST_ALL) return;  // the rest is the first block's alone
    if (route == LIST_ALL && s.list_n <= kShort) {
      // A short list: every element against every other, eight lanes an element,
      // gives its rank and the weight in front of it, by value and then by index,
      // with two barriers instead of a search each.
      const int n = s.list_n, i = tid >> 3, part = tid & 7;
      u64* ms = reinterpret_cast<u64*>(s.n);
      const uint2 e = i < n ? list[i] : make_uint2(0u, 0u);
      const double w = R.weight(e.x);
      const u64 m = i < n ? R.fixed(w) : 0ull;
      if (i < n && part == 0) ms[i] = m;
      __syncthreads();
      int above = 0;
      u64 front = 0ull;
      if (i < n)
        for (int j = part; j < n; j += 8) {
          const uint2 f = list[j];
          above += f.x > e.x;
          front += f.x > e.x || (f.x == e.x && f.y < e.y) ? ms[j] : 0ull;
        }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        above += __shfl_xor_sync(0xffffffffu, above, o);
        front += __shfl_xor_sync(0xffffffffu, front, o);
      }
      bool in = i < n && (!by_count || above < want_k);
      if (by_mass) {
        if (by_count) total = R.block_sum(in && part == 0 ? m : 0ull);
        in = in && front <= (u64)floor(fmax(p, 0.0) * (double)total);
      }
      const u64 mine = in && w >= least ? m : 0ull;
      const u64 all = R.block_sum(part == 0 ? mine : 0ull);  // (and every thread has read ms)
      if (i < n && part == 0) ms[i] = mine;
      __syncthreads();
      const u64 goal = min((u64)floor(fmax(u, 0.0) * (double)all), all - 1ull);
      u64 run = 0ull;
      if (i < n)
        for (int j = part; j < n; j += 8) run += list[j].y < e.y ? ms[j] : 0ull;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) run += __shfl_xor_sync(0xffffffffu, run, o);
      if (part == 0 && mine && run <= goal && goal < run + mine) {
        a.token[row] = (int64_t)e.y;
        a.logprob[row] =
            (float)((e.x == R.top_key ? 0.0 : (double)value_of(e.x) - R.zmax) - log((double)all / s.table[0]));
      }
      return;
    }
    if (rank == 0) {
      R.listed = route == LIST_ALL || route == LIST_BORDER;
      if (by_count) {
        threshold = open ? R.template narrow<false>(lo, hi, want, ahead, ties_n, false) : lo;
        if (by_mass) {
          lo = threshold;
          hi = R.top_key;
          u64 m = 0ull;
          R.each([&](uint32_t key, int) {
            if (key >= lo) m += R.fixed(R.weight(key));
          });
          total = R.block_sum(m);
          want = (u64)floor(fmax(p, 0.0) * (double)total);
        }
      }
      if (by_mass) {
        ahead = 0ull;
        if (!by_count && R.listed)
          for (int r = 0; r < blocks; ++r) ahead += s.total[r];
        threshold = R.template narrow<true>(lo, hi, want, ahead, ties_n, !by_count && !R.listed);
        if (ties_n > 1) {
          ties_in = (want - ahead) / R.fixed(R.weight(threshold)) + 1ull;  // weight > 0: the sum crosses within these ties
          if (ties_in >= ties_n) ties_in = ~0ull;
        }
      }
    }
  }
  // of the threshold's ties those up to this index
  if (ties_in != ~0ull) {  // (the first block alone comes here)
    __syncthreads();
    R.template clear<false>();
    R.each([&](uint32_t key, int i) {
      if (key == threshold) atomicAdd(&s.n[i >> ish], 1u);
    });
    R.template find<false>(0ull, ties_in);
    const int i = (s.bin << ish) + tid;
    const bool tie = tid < (1 << ish) && i < a.V && R.key_at(i) == threshold;
    const u64 base = s.ahead;
    u64 all;
    const u64 before = base + R.block_before(tie ? 1ull : 0ull, all);
    if (tie && before + 1ull == ties_in) s.at = i;
    __syncthreads();
    tie_last = s.at;
  }
  auto kept = [&](uint32_t key, int i) -> u64 {
    const double w = R.weight(key);
    const bool in = key >= threshold && key >= min_cut && !(key == threshold && i > tie_last) && w >= least;
    return in ? R.fixed(w) : 0ull;
  };
  // 4. the draw: kept weight by index
  if (route == LIST_ALL) {
    __syncthreads();
    R.template clear<true>();
    R.each([&](uint32_t key, int i) {
      const u64 m = kept(key, i);
      if (m) R.add_mass(i >> ish, m);
    });
    __syncthreads();
  } else {
    if (filtered) {
      if (rank == 0) {
        __syncthreads();
        R.template clear<true>();
        if (tid == 0) {
          s.threshold = threshold;
          s.tie_last = tie_last;
        }
      }
      R.cluster_sync(blocks);
      if (rank > 0) {
        threshold = first.threshold;
        tie_last = first.tie_last;
      }
    }
    const uint32_t from = max(threshold, min_cut);
    const float cut = value_of(from);
    // a vector lies in one index bin, and a warp's vectors follow one another
    const bool aligned = ish >= 2 && (i0 & (VEC - 1)) == 0;
    const bool everything = from <= kLowest;
    R.groups(i0, i1, [&](const float (&z)[VEC], int i, int n) {
      bool hit = everything;
#pragma unroll
      for (int k = 0; k < VEC; ++k) hit |= k < n && z[k] >= cut;
      if (!__any_sync(0xffffffffu, hit)) return;
      u64 m = 0ull;
#pragma unroll
      for (int k = 0; k < VEC; ++k)
      {
        u64 w = kept(R.key_or_low(z[k]), i + k);
        w = k < n ? w : 0ull;
        if (!aligned && w) R.add_mass((i + k) >> ish, w);
        m += w;
      }
      if (aligned) R.add_by_index(i, m);  // by every lane
    });
    __syncthreads();
    if (rank > 0) {  // the bins of a block's part are its own
      const int b = (i0 >> ish) + tid;
      if (i0 < i1 && b <= (i1 - 1) >> ish) {
        first.m0[b] = s.m0[b];
        first.m1[b] = s.m1[b];
        first.m2[b] = s.m2[b];
      }
    }
    R.cluster_sync(blocks);
    if (rank > 0) return;
  }
  u64 sum = R.bin_mass(tid), all;
  const u64 run = R.block_before(sum, all);
  // run > u * total for the integer run means run > floor(u * total); u = 1 ends at the last kept token
  const u64 goal = min((u64)floor(fmax(u, 0.0) * (double)all), all - 1ull);
  if (run <= goal && run + sum > goal) {
    s.bin = tid;
    s.ahead = run;
  }
  __syncthreads();
  {
    const int i = (s.bin << ish) + tid;
    const bool on = tid < (1 << ish) && i < a.V;
    const uint32_t key = on ? R.key_at(i) : 0u;
    const u64 m = kept(key, i);
    u64 ignored;
    const u64 base = s.ahead;
    const u64 in_front = base + R.block_before(m, ignored);
    if (on && in_front <= goal && in_front + m > goal) {
      a.token[row] = i;
      a.logprob[row] = (float)((key == R.top_key ? 0.0 : (double)value_of(key) - R.zmax) - log((double)all / s.table[0]));
    }
  }
}

template <typename T>
void launch_sample(const SampleArgs& a, int64_t B, int cluster, size_t smem) {
  C10_CUDA_CHECK(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedLimit));
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
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, sample_kernel<T>, a));
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
  TORCH_CHECK(logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1), what, ": logits must be [B, V] with contiguous rows");
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
                    seen->size(0) == B && (seen->stride(1) == 1 || seen->size(1) == 1) && seen->size(1) < (1ll << 31),
                what, ": generated must be int64 [", B, ", n] with contiguous rows on the logits' device");
    a.seen = seen->data_ptr<int64_t>();
    a.seen_s = seen->stride(0);
    a.L = (int)seen->size(1);
  }
  TORCH_CHECK(B < (1ll << 28), what, ": too many rows in one call");
  int bits = 15;
  while ((1ll << bits) < V) ++bits;
  a.limb = std::min(16, 32 - bits);  // V limbs of this width sum to less than 2^32
  a.fbits = std::min(62 - bits, 3 * a.limb - 1);
  while ((V - 1) >> a.index_shift >= kBins) ++a.index_shift;
  // blocks that help with the two passes over a row, while SMs are free and a part is worth their barriers
  int cluster = 1;
  while (cluster < 8 && B * cluster * 2 <= num_sms() && V / (cluster * 2) >= 2048) cluster *= 2;
  a.slice = (int)((V + cluster - 1) / cluster);
  if (cluster > 1) a.slice = (((a.slice - 1) >> a.index_shift) + 1) << a.index_shift;  // whole index bins, of 4 or more
  const size_t fixed = sizeof(Shared) + (a.seen ? ((V + 31) / 32 + 3) / 4 * 16 : 0);
  a.list_cap = (int)std::min<int64_t>(V, (int64_t)(kSharedLimit - fixed) / 8);
  const size_t smem = fixed + (size_t)a.list_cap * 8;
  TB_DISPATCH_FLOAT(logits.scalar_type(), what, [&] { launch_sample<scalar_t>(a, B, cluster, smem); });
  check_launch(what);
  return {token, logprob};
}

}  // namespace tb
