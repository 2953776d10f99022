// Token sampling: temperature, repetition penalty, top-k, top-p, min-p and the
// draw itself, from uniform numbers that the caller gives, one row per request.
//
//   z_i = logit_i / T            (fp32; then / penalty for tokens already seen; NaN = -inf)
//   w_i = exp(z_i - max z)       (fp64)
//   top-k:  keep z_i >= the k-th largest z (all ties with it)
//   top-p:  in descending order (ties: lower index first) keep i while the
//           weight in front of it is <= p * sum of the weights left by top-k
//   min-p:  keep w_i >= min_p
//   token:  the first i, by index, whose running sum of kept weights exceeds
//           u * (their sum)
// T <= 0 takes the first largest z.  Weights and sums are fp64: a token sits on
// the border of a running sum, and fp32 would move it.
#include "common.cuh"

namespace tb {
namespace {

constexpr int kThreads = 1024;

// one value for every row, or one per row
struct Setting {
  const float* per_row;
  float all;
  __device__ __forceinline__ float at(int row) const { return per_row ? per_row[row] : all; }
};

struct SampleArgs {
  const void* logits;
  int64_t ls;
  int V;
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

template <typename T> __device__ __forceinline__ T block_reduce_sum(T v, T* red) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) red[wid] = v;
  __syncthreads();
  v = red[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  extern __shared__ uint32_t seen_bits[];
  __shared__ double red_d[32];
  __shared__ long long red_l[32];
  __shared__ uint32_t red_u[32];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const T* lr = (const T*)a.logits + row * a.ls;
  const float temp = a.temp.at(row);
  const bool greedy = !(temp > 0.f);
  const float div = greedy ? 1.f : temp, pen = a.penalty.at(row);
  if (a.seen) {
    for (int i = tid; i < (a.V + 31) / 32; i += kThreads) seen_bits[i] = 0u;
    __syncthreads();
    for (int i = tid; i < a.L; i += kThreads) {
      const int64_t t = a.seen[row * a.seen_s + i];
      if (t >= 0 && t < a.V) atomicOr(&seen_bits[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
  }
  auto key_at = [&](int i) -> uint32_t {
    float z = __fdiv_rn(to_f<T>(lr[i]), div);
    if (a.seen && (seen_bits[i >> 5] >> (i & 31) & 1u)) z = __fdiv_rn(z, pen);
    return isnan(z) ? key_of(-INFINITY) : key_of(z == 0.f ? 0.f : z);
  };
  // largest key, lowest index
  uint32_t best = 0;
  int best_i = 0x7fffffff;
  for (int i = tid; i < a.V; i += kThreads) {
    const uint32_t k = key_at(i);
    if (k > best || (k == best && i < best_i)) { best = k; best_i = i; }
  }
  long long packed = ((long long)best << 31) | (0x7fffffff - best_i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) packed = max(packed, __shfl_xor_sync(0xffffffffu, packed, o));
  if (lane == 0) red_l[wid] = packed;
  __syncthreads();
  packed = red_l[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) packed = max(packed, __shfl_xor_sync(0xffffffffu, packed, o));
  const uint32_t top_key = (uint32_t)(packed >> 31);
  const int top_i = 0x7fffffff - (int)(packed & 0x7fffffff);
  const float zmax = value_of(top_key);
  if (greedy || zmax == -INFINITY) {
    if (tid == 0) {
      a.token[row] = top_i;
      a.logprob[row] = greedy ? 0.f : __int_as_float(0x7fffffff);
    }
    return;
  }
  auto weight = [&](uint32_t k) -> double {
    if (k == top_key) return 1.0;
    return exp((double)value_of(k) - (double)zmax);
  };
  // top-k: the largest threshold that at least k keys reach
  uint32_t kth = 0;
  const int64_t want = (a.top_k ? a.top_k[row] : a.top_k0);
  if (want > 0 && want < a.V) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = kth | (1u << bit);
      int n = 0;
      for (int i = tid; i < a.V; i += kThreads) n += key_at(i) >= t;
      n = block_reduce_sum<long long>(n, red_l);
      if (n >= want) kth = t;
    }
  }
  // top-p: the smallest key whose weight in front is within the nucleus
  uint32_t pth = kth;
  int64_t ties = a.V;  // how many keys equal to pth are kept
  const double p = (double)a.top_p.at(row);
  if (p < 1.0) {
    double s = 0.0;
    for (int i = tid; i < a.V; i += kThreads) {
      const uint32_t k = key_at(i);
      if (k >= kth) s += weight(k);
    }
    const double nucleus = p * block_reduce_sum(s, red_d);
    // keys above t weigh <= nucleus  <=>  t itself is kept; find the smallest such t
    uint32_t lo = kth, hi = top_key;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      double above = 0.0;
      for (int i = tid; i < a.V; i += kThreads) {
        const uint32_t k = key_at(i);
        if (k > mid) above += weight(k);
      }
      above = block_reduce_sum(above, red_d);
      if (above <= nucleus) hi = mid; else lo = mid + 1;
    }
    pth = lo;
    // pth need not be a present key; if it is, some of its ties may fall out
    double above = 0.0;
    long long n = 0;
    for (int i = tid; i < a.V; i += kThreads) {
      const uint32_t k = key_at(i);
      if (k > pth) above += weight(k);
      n += k == pth;
    }
    above = block_reduce_sum(above, red_d);
    n = block_reduce_sum(n, red_l);
    if (n > 0) {
      const double w = weight(pth);
      ties = w > 0.0 ? (int64_t)fmin(floor((nucleus - above) / w) + 1.0, (double)a.V) : a.V;
      if (ties < 1) ties = 1;
    }
  }
  // kept weights by index: contiguous chunks per thread
  const double least = (double)a.min_p.at(row);
  const int per = (a.V + kThreads - 1) / kThreads;
  const int i0 = min(tid * per, a.V), i1 = min(i0 + per, a.V);
  // rank of a key equal to pth among its ties: exclusive scan of tie counts
  int tie_base = 0;
  if (ties < a.V) {
    int n = 0;
    for (int i = i0; i < i1; ++i) n += key_at(i) == pth;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) red_u[wid] = incl;
    __syncthreads();
    int base = 0;
    for (int x = 0; x < wid; ++x) base += red_u[x];
    tie_base = base + incl - n;
  }
  auto kept = [&](uint32_t k, int& tie) -> double {
    if (k < pth || k < kth) return 0.0;
    if (k == pth && tie++ >= ties) return 0.0;
    const double w = weight(k);
    return w >= least ? w : 0.0;
  };
  double mine = 0.0;
  int tie = tie_base;
  for (int i = i0; i < i1; ++i) mine += kept(key_at(i), tie);
  double incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  __syncthreads();
  if (lane == 31) red_d[wid] = incl;
  __syncthreads();
  double base = 0.0, total = 0.0;
  for (int x = 0; x < 32; ++x) {
    if (x == wid) base = total;
    total += red_d[x];
  }
  base += incl - mine;
  const double target = (double)a.u[row] * total;
  __shared__ int hit;
  if (tid == 0) hit = 0x7fffffff;
  __syncthreads();
  // the first index whose running sum exceeds the target; u = 1 ends at the last kept one
  double run = base;
  tie = tie_base;
  int last = -1;
  for (int i = i0; i < i1; ++i) {
    const double w = kept(key_at(i), tie);
    run += w;
    if (w > 0.0) {
      last = i;
      if (run > target) {
        atomicMin(&hit, i);
        break;
      }
    }
  }
  __syncthreads();
  __shared__ int last_kept;
  if (tid == 0) last_kept = -1;
  __syncthreads();
  if (hit == 0x7fffffff && last >= 0) atomicMax(&last_kept, last);
  __syncthreads();
  if (tid == 0) {
    const int t = hit != 0x7fffffff ? hit : last_kept;
    a.token[row] = t;
    a.logprob[row] = (float)log(weight(key_at(t)) / total);
  }
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
  TORCH_CHECK(V >= 1 && V <= (1 << 20), what, ": a vocabulary of 1 to 2^20 tokens");
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
  const size_t smem = a.seen ? (V + 31) / 32 * 4 : 0;
  TB_DISPATCH_FLOAT(logits.scalar_type(), what, [&] {
    if (smem > 32 * 1024)
      C10_CUDA_CHECK(cudaFuncSetAttribute(sample_kernel<scalar_t>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          160 * 1024));
    sample_kernel<scalar_t><<<(unsigned)B, kThreads, smem, stream()>>>(a);
  });
  check_launch(what);
  return {token, logprob};
}

}  // namespace tb
