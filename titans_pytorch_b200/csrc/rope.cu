// Rotary positions, forward and backward (the same rotation by the opposite
// angle).  x [B, T, H, d] with any strides over B, T, H; the first 2n of d are
// rotated in pairs, interleaved (2i, 2i+1) or half (i, i+n), the rest copied.
//
// x is read once and y written once.  A block takes a few tokens; their cos /
// sin are computed once in shared memory (fp64 angle, see rope.cuh) and serve
// every head, then each thread moves 16-byte vectors.  Half layout, fp32 (1 x
// 16384 x 32 x 96): 74 us for 403 MB, 83 % of the copy rate, bound by memory.
// Interleaved, bf16 (8 x 4096 x 24 x 64): 43.5 us for 201 MB, 71 %; there the
// instructions of eight elements a vector weigh as much as the memory.
#include "common.cuh"
#include "rope.cuh"

namespace tb {
namespace {

struct RopeArgs {
  const void* x;
  void* y;
  const int64_t* pos;
  const float* freq;
  int64_t sxb, sxt, sxh, spb, spt;
  int64_t tokens;  // B * T
  int T, H, d, n;
  float amplitude, sign;
  FastDiv by_token, by_head, by_t, by_pair;  // work items of a token, of a head; T; pairs of a token
};

constexpr int kThreads = 256;

// Interleaved: a 16-byte vector holds whole pairs; the table is padded past the
// rotated part, and what is not rotated there is put back as it was (times (1, 0)
// an infinity would spoil the other of its pair, and -0 its sign).
// Half: a work item is a pair of vectors (i, i + n) or one vector of the tail.
//
// The vectors are requested before the table is computed, so that the loads
// and the fp64 angles wait at the same time.
template <typename T, bool HALF>
__global__ void __launch_bounds__(kThreads) rope_vec_kernel(RopeArgs a, int tok_per_block) {
  constexpr int V = Vec16<T>::N, ITEMS = HALF ? 2 : 4;  // work items a thread has in flight
  extern __shared__ __align__(16) float tab_raw[];         // cos [tok_per_block][pairs], then sin
  float* tab = tab_raw;
  const int pairs = HALF ? a.n : a.d / 2;
  const int tok0 = blockIdx.x * tok_per_block;
  const int toks = (int)min((int64_t)tok_per_block, a.tokens - tok0);
  const int rot = a.n / V, head_items = HALF ? rot + (a.d - 2 * a.n) / V : a.d / V;
  const int tok_items = a.H * head_items, items = toks * tok_items;
  struct Item {
    uint4 x, y;
    T* dst;
    int t, v;
  } it[ITEMS];
  auto fetch = [&](int base) {
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) {
      const int i = base + q * kThreads + threadIdx.x;
      if (i < items) {
        int rem, v, tt;
        const int t = a.by_token(i, rem), h = a.by_head(rem, v);
        const int tok = tok0 + t, b = a.by_t(tok, tt);
        const T* x = (const T*)a.x + b * a.sxb + tt * a.sxt + h * a.sxh;
        it[q].dst = (T*)a.y + ((int64_t)tok * a.H + h) * a.d;
        it[q].t = t;
        it[q].v = v;
        const int at = HALF && v >= rot ? 2 * a.n + (v - rot) * V : v * V;
        it[q].x = *reinterpret_cast<const uint4*>(x + at);
        if (HALF && v < rot) it[q].y = *reinterpret_cast<const uint4*>(x + a.n + at);
      }
    }
  };
  fetch(0);
  for (int i = threadIdx.x; i < toks * pairs; i += kThreads) {
    int p, tt;
    const int t = a.by_pair(i, p);
    const int tok = tok0 + t, b = a.by_t(tok, tt);
    float2 cs = make_float2(1.f, 0.f);
    if (p < a.n) {
      cs = rope_cos_sin(a.pos[b * a.spb + tt * a.spt], a.freq[p], a.amplitude);
      cs.y *= a.sign;
    }
    tab[i] = cs.x;
    tab[tok_per_block * pairs + i] = cs.y;
  }
  __syncthreads();
  for (int base = 0; base < items; base += ITEMS * kThreads) {
    if (base) fetch(base);
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) {
      if (base + q * kThreads + (int)threadIdx.x >= items) break;
      const float* cs = tab + it[q].t * pairs;
      const float* sn = cs + tok_per_block * pairs;
      const int v = it[q].v;
      Vec16<T> x, y;
      x.raw = it[q].x;
      if constexpr (HALF) {
        if (v < rot) {
          y.raw = it[q].y;
          float u[V], w[V], c[V], n[V];
          table_load(cs + v * V, c);
          table_load(sn + v * V, n);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float p0 = to_f<T>(x.v[k]), p1 = to_f<T>(y.v[k]);
            u[k] = p0 * c[k] - p1 * n[k];
            w[k] = p0 * n[k] + p1 * c[k];
          }
          store16<T>(it[q].dst + v * V, u);
          store16<T>(it[q].dst + a.n + v * V, w);
        } else {
          *reinterpret_cast<uint4*>(it[q].dst + 2 * a.n + (v - rot) * V) = it[q].x;
        }
      } else {
        float u[V], c[V / 2], n[V / 2];
        table_load(cs + v * (V / 2), c);
        table_load(sn + v * (V / 2), n);
#pragma unroll
        for (int k = 0; k < V; k += 2) {
          const float p0 = to_f<T>(x.v[k]), p1 = to_f<T>(x.v[k + 1]);
          u[k] = p0 * c[k / 2] - p1 * n[k / 2];
          u[k + 1] = p0 * n[k / 2] + p1 * c[k / 2];
        }
#pragma unroll
        for (int k = 0; k < V; ++k) y.v[k] = from_f<T>(u[k]);
        const int live = 2 * a.n - v * V;  // elements of the vector that are rotated
        if (live < V)
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (k >= live) y.v[k] = x.v[k];
        *reinterpret_cast<uint4*>(it[q].dst + v * V) = y.raw;
      }
    }
  }
}

// Any size, stride and alignment: one element pair (or one tail element) per item.
template <typename T>
__global__ void __launch_bounds__(kThreads) rope_scalar_kernel(RopeArgs a, bool half, int64_t sxd) {
  extern __shared__ __align__(16) float tab_raw[];
  float2* tab = reinterpret_cast<float2*>(tab_raw);
  const int tok = blockIdx.x;
  const int b = tok / a.T, tt = tok - b * a.T;
  for (int p = threadIdx.x; p < a.n; p += kThreads) {
    float2 cs = rope_cos_sin(a.pos[b * a.spb + tt * a.spt], a.freq[p], a.amplitude);
    cs.y *= a.sign;
    tab[p] = cs;
  }
  __syncthreads();
  const int head_items = a.d - a.n;
  for (int i = threadIdx.x; i < a.H * head_items; i += kThreads) {
    const int h = i / head_items, v = i - h * head_items;
    const T* x = (const T*)a.x + b * a.sxb + tt * a.sxt + h * a.sxh;
    T* y = (T*)a.y + ((int64_t)tok * a.H + h) * a.d;
    if (v < a.n) {
      const int i0 = half ? v : 2 * v, i1 = half ? v + a.n : 2 * v + 1;
      const float p = to_f<T>(x[i0 * sxd]), q = to_f<T>(x[i1 * sxd]);
      const float2 c = tab[v];
      y[i0] = from_f<T>(p * c.x - q * c.y);
      y[i1] = from_f<T>(p * c.y + q * c.x);
    } else {
      y[v + a.n] = x[(v + a.n) * sxd];
    }
  }
}

}  // namespace

at::Tensor rotary_embedding(const at::Tensor& x, const at::Tensor& pos, const at::Tensor& freq, bool half,
                            double amplitude, bool backward) {
  TB_CHECK_CUDA(x);
  TORCH_CHECK(x.dim() == 4, "rotary_embedding: x must be [B, T, H, d]");
  TORCH_CHECK(pos.device() == x.device() && freq.device() == x.device(),
              "rotary_embedding: x, positions and inv_freq must be on one device");
  TORCH_CHECK(pos.scalar_type() == at::kLong && freq.scalar_type() == at::kFloat && freq.dim() == 1 &&
                  freq.is_contiguous(),
              "rotary_embedding: int64 positions and a contiguous fp32 inv_freq");
  const int64_t B = x.size(0), T = x.size(1), H = x.size(2), d = x.size(3), n = freq.numel();
  TORCH_CHECK(2 * n <= d, "rotary_embedding: ", n, " frequencies rotate ", 2 * n, " of only ", d, " dimensions");
  TORCH_CHECK(d <= 1024 && H <= (1 << 20) && T < (1ll << 31), "rotary_embedding: at most 1024 dimensions a head");
  TORCH_CHECK((pos.dim() == 1 && pos.size(0) == T) || (pos.dim() == 2 && pos.size(0) == B && pos.size(1) == T),
              "rotary_embedding: positions must be [T] or [B, T]");
  const at::cuda::CUDAGuard g(x.device());
  at::Tensor y = at::empty({B, T, H, d}, x.options());
  if (y.numel() == 0) return y;
  RopeArgs a;
  a.x = x.data_ptr();
  a.y = y.data_ptr();
  a.pos = pos.data_ptr<int64_t>();
  a.freq = freq.data_ptr<float>();
  a.sxb = x.stride(0);
  a.sxt = x.stride(1);
  a.sxh = x.stride(2);
  a.spb = pos.dim() == 2 ? pos.stride(0) : 0;
  a.spt = pos.stride(-1);
  a.tokens = B * T;
  TORCH_CHECK(a.tokens < (1ll << 31), "rotary_embedding: too many tokens in one call");
  a.T = (int)T;
  a.H = (int)H;
  a.d = (int)d;
  a.n = (int)n;
  a.amplitude = (float)amplitude;
  a.sign = backward ? -1.f : 1.f;
  TB_DISPATCH_FLOAT(x.scalar_type(), "rotary_embedding", [&] {
    constexpr int V = Vec16<scalar_t>::N;
    const bool vec = (x.stride(3) == 1 || d == 1) && d % V == 0 && aligned16(x) && a.sxb % V == 0 &&
                     a.sxt % V == 0 && a.sxh % V == 0 && (!half || n % V == 0);
    if (!vec) {
      rope_scalar_kernel<scalar_t><<<(unsigned)a.tokens, kThreads, n * sizeof(float2), stream()>>>(a, half,
                                                                                                x.stride(3));
      return;
    }
    // enough tokens a block for two rounds of its loads, if that still fills the GPU: the table's latency is
    // paid once a block (one round 46, two 43.5, four 46 us for 8 x 4096 x 24 x 64 bf16)
    const int64_t items = half ? H * (n / V + (d - 2 * n) / V) : H * d / V;
    int64_t per = std::max<int64_t>(1, 2 * (half ? 2 : 4) * kThreads / std::max<int64_t>(items, 1));
    per = std::min(per, std::max<int64_t>(1, a.tokens / (num_sms() * 4)));
    const int64_t pair_bytes = (half ? std::max<int64_t>(n, 1) : d / 2) * sizeof(float2);
    per = std::min<int64_t>({per, 16, 48 * 1024 / pair_bytes});
    a.by_token = FastDiv((uint32_t)std::max<int64_t>(items, 1));
    a.by_head = FastDiv((uint32_t)std::max<int64_t>(items / H, 1));
    a.by_t = FastDiv((uint32_t)T);
    a.by_pair = FastDiv((uint32_t)std::max<int64_t>(half ? n : d / 2, 1));
    const size_t smem = per * pair_bytes;
    const unsigned blocks = (unsigned)((a.tokens + per - 1) / per);
    if (half)
      rope_vec_kernel<scalar_t, true><<<blocks, kThreads, smem, stream()>>>(a, (int)per);
    else
      rope_vec_kernel<scalar_t, false><<<blocks, kThreads, smem, stream()>>>(a, (int)per);
  });
  check_launch("rotary_embedding");
  return y;
}

}  // namespace tb
