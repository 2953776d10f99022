// The key/value cache: new tokens are rotated, quantised and stored in one
// pass, and stored tokens read back in order.
//
// Slot of a token = its position modulo the number of slots (a ring; a linear
// cache is a ring that never wraps).  The 8-bit kinds keep one fp32 scale per
// (token, head): with amax the largest magnitude of the row and top = 127
// (int8) or 448 (e4m3),
//     stored = round(x * (top / amax)),  scale = amax / top,
// x in fp32 after the rotation; rounding to the nearest, ties to even.  Rows
// with amax < 2^-100 are stored as zeros (top / amax would overflow); a row
// with an infinity or NaN gets the scale NaN, so it reads back as NaN instead
// of as plausible numbers.
//
// Bound by memory: each new row is read once (a half-layout row finds its
// partner elements in L1) and written once.
#include "kv_cache.cuh"
#include "rope.cuh"

namespace tb {
namespace {

constexpr int kThreads = 256;

struct Rows {  // [B, T, H, d], last dimension contiguous
  const void* p;
  int64_t sb, st, sh;
  int H;
};

struct WriteArgs {
  Rows k, v, q;
  CacheView ck, cv;
  void* q_out;
  const int64_t* start;
  const int64_t* count;  // or null: all T
  const float* freq;
  int64_t start_s, count_s, offset;
  int T, S, d, n;
  float amplitude;
  int half;
};

// 8 elements of row x from column c, rotated.  tab: cos / sin of the token's pairs.
template <typename T>
__device__ __forceinline__ void rotated8(const T* x, int c, const float2* tab, int n, bool half, float (&v)[8]) {
  load8<T>(x + c, v);
  if (c >= 2 * n) return;
  if (!half) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const int p = (c + i) >> 1;
      if (p < n) {
        const float2 cs = tab[p];
        const float a = v[i], b = v[i + 1];
        v[i] = a * cs.x - b * cs.y;
        v[i + 1] = a * cs.y + b * cs.x;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = c + i;
      if (j < n) {
        const float2 cs = tab[j];
        v[i] = v[i] * cs.x - to_f<T>(x[j + n]) * cs.y;
      } else if (j < 2 * n) {
        const float2 cs = tab[j - n];
        v[i] = to_f<T>(x[j - n]) * cs.y + v[i] * cs.x;
      }
    }
  }
}

// Block = one token of one sequence, all its heads: first the token's cos /
// sin, then LANES lanes per row (a power of two >= d / 8), 8 elements a lane.
template <typename T, typename C, int LANES>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(WriteArgs a) {
  extern __shared__ float2 tab[];  // [n]
  const int t = blockIdx.x, b = blockIdx.y;
  const int64_t start = a.start[b * a.start_s];
  int64_t count = a.count ? a.count[b * a.count_s] : a.T;
  count = min(max(count, (int64_t)0), (int64_t)a.T);
  const int64_t pos = start + t;
  // a token that a later one of this call would overwrite is not stored, nor one before position 0
  const bool stored = t < count && t >= count - a.S && pos >= 0;
  if (!stored && a.q.p == nullptr) return;
  for (int p = threadIdx.x; p < a.n; p += kThreads) tab[p] = rope_cos_sin(pos + a.offset, a.freq[p], a.amplitude);
  __syncthreads();
  const int slot = stored ? (int)(pos % a.S) : 0;
  const int lane = threadIdx.x % LANES;
  const int c = lane * 8;
  const bool on = c < a.d;
  const int rows = a.q.H + (stored ? a.k.H + a.v.H : 0);
  // whole warps stay in the loop for the shuffles
  for (int r0 = 0; r0 < rows; r0 += kThreads / LANES) {
    const int r = r0 + threadIdx.x / LANES;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r < a.q.H) {
      if (on) {
        const T* src = (const T*)a.q.p + b * a.q.sb + t * a.q.st + r * a.q.sh;
        rotated8<T>(src, c, tab, a.n, a.half, x);
        store8<T>((T*)a.q_out + (((int64_t)b * a.T + t) * a.q.H + r) * a.d + c, x);
      }
    }
    const int kv = r - a.q.H;
    const bool mine = kv >= 0 && r < rows;
    const bool is_v = kv >= a.k.H;
    const int h = is_v ? kv - a.k.H : kv;
    if (mine && on) {
      const Rows& in = is_v ? a.v : a.k;
      const T* src = (const T*)in.p + b * in.sb + t * in.st + h * in.sh;
      if (is_v)
        load8<T>(src + c, x);
      else
        rotated8<T>(src, c, tab, a.n, a.half, x);
    }
    const CacheView& dst = is_v ? a.cv : a.ck;
    if constexpr (CacheTraits<C>::scaled) {
      float amax = 0.f;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        amax = fmaxf(amax, fabsf(x[i]));
        bad |= !isfinite(x[i]);
      }
      int bad_any = bad;
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        bad_any |= __shfl_xor_sync(0xffffffffu, bad_any, o);
      }
      constexpr float top = CacheTraits<C>::top;
      const bool full = amax >= 7.888609052210118e-31f && !bad_any;  // 2^-100
      const float inv = full ? top / amax : 0.f;
      float scale = full ? amax / top : 1.f;
      if (bad_any) scale = __int_as_float(0x7fffffff);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = bad_any ? 0.f : x[i] * inv;
      if (mine && lane == 0) dst.scale[b * dst.qb + h * dst.qh + slot * dst.qs] = scale;
    }
    if (mine && on) store8<C>((C*)dst.data + b * dst.sb + h * dst.sh + slot * dst.ss + c, x);
  }
}

struct ReadArgs {
  CacheView ck, cv;
  void* ko;
  void* vo;
  const int64_t* lengths;
  int64_t len_s;
  int H, S, n, d;
};

// Row i of the output: the i-th of the newest min(length, slots, n) tokens, in
// order; zeros behind the last.  Block = rows_per_block rows of one (sequence,
// head, keys or values); one thread moves 8 elements.
template <typename C, typename T>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(ReadArgs a) {
  const int per_row = a.d / 8;
  const int64_t i64 = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int h = blockIdx.y % a.H, b = blockIdx.y / a.H;
  const int i = (int)(i64 / per_row), c = (int)(i64 - (int64_t)i * per_row) * 8;
  if (i >= a.n) return;
  const bool is_v = blockIdx.z;
  const CacheView& src = is_v ? a.cv : a.ck;
  const int64_t len = max(a.lengths[b * a.len_s], (int64_t)0);
  const int64_t held = min(len, (int64_t)min(a.S, a.n));
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (i < held) {
    const int64_t slot = (len - held + i) % a.S;
    load8<C>((const C*)src.data + b * src.sb + h * src.sh + slot * src.ss + c, x);
    if constexpr (CacheTraits<C>::scaled) {
      const float s = src.scale[b * src.qb + h * src.qh + slot * src.qs];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] *= s;
    }
  }
  T* dst = (T*)(is_v ? a.vo : a.ko);
  store8<T>(dst + ((int64_t)blockIdx.y * a.n + i) * a.d + c, x);
}

// `hold` keeps the copy that unaligned rows need.
Rows rows_of(const at::Tensor& x, at::Tensor& hold, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 4, what, ": new tokens must be CUDA tensors [B, T, H, d]");
  const at::cuda::CUDAGuard g(x.device());
  const int64_t size = x.element_size();
  const bool fits = x.stride(3) == 1 && x.stride(0) * size % 16 == 0 && x.stride(1) * size % 16 == 0 &&
                    x.stride(2) * size % 16 == 0 && aligned16(x);
  hold = fits ? x : contig16(x);
  return Rows{hold.data_ptr(), hold.stride(0), hold.stride(1), hold.stride(2), (int)hold.size(2)};
}

template <typename T, typename C>
void launch_write(const WriteArgs& a, int64_t B) {
  const dim3 grid((unsigned)a.T, (unsigned)B);
  const size_t smem = a.n * sizeof(float2);
  if (a.d <= 64)
    kv_write_kernel<T, C, 8><<<grid, kThreads, smem, stream()>>>(a);
  else if (a.d <= 128)
    kv_write_kernel<T, C, 16><<<grid, kThreads, smem, stream()>>>(a);
  else
    kv_write_kernel<T, C, 32><<<grid, kThreads, smem, stream()>>>(a);
}

}  // namespace

at::Tensor kv_cache_write(at::Tensor& ck, at::Tensor& cv, const c10::optional<at::Tensor>& ks,
                          const c10::optional<at::Tensor>& vs, const at::Tensor& k, const at::Tensor& v,
                          const at::Tensor& start, const c10::optional<at::Tensor>& count,
                          const c10::optional<at::Tensor>& q, const c10::optional<at::Tensor>& freq, bool half,
                          double amplitude, int64_t offset) {
  const char* what = "kv_cache_write";
  WriteArgs a{};
  a.ck = cache_view(ck, ks, what);
  a.cv = cache_view(cv, vs, what);
  TORCH_CHECK(ck.sizes() == cv.sizes() && ck.scalar_type() == cv.scalar_type() && ck.device() == cv.device(), what,
              ": the key and value caches must have one shape, type and device");
  at::Tensor hold_k, hold_v, hold_q;
  a.k = rows_of(k, hold_k, what);
  a.v = rows_of(v, hold_v, what);
  const int64_t B = ck.size(0), H = ck.size(1), d = ck.size(3), T = k.size(1);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(2) == H && k.size(3) == d &&
                  k.scalar_type() == v.scalar_type() && k.device() == ck.device() && v.device() == ck.device(),
              what, ": new keys and values must be [", B, ", T, ", H, ", ", d, "] of one type on the cache's device");
  TORCH_CHECK(start.device() == ck.device() && start.scalar_type() == at::kLong && start.dim() == 1 &&
                  start.size(0) == B, what, ": start must be int64 [", B, "] on the cache's device");
  TORCH_CHECK(B < 65536 && T < (1ll << 31), what, ": at most 65535 sequences in one call");
  const at::cuda::CUDAGuard g(ck.device());
  a.start = start.data_ptr<int64_t>();
  a.start_s = start.stride(0);
  if (count.has_value() && count->defined()) {
    TORCH_CHECK(count->device() == ck.device() && count->scalar_type() == at::kLong && count->dim() == 1 &&
                    count->size(0) == B, what, ": counts must be int64 [", B, "] on the cache's device");
    a.count = count->data_ptr<int64_t>();
    a.count_s = count->stride(0);
  }
  at::Tensor q_out;
  if (q.has_value() && q->defined()) {
    a.q = rows_of(*q, hold_q, what);
    TORCH_CHECK(q->size(0) == B && q->size(1) == T && q->size(3) == d && q->scalar_type() == k.scalar_type() &&
                    q->device() == ck.device(),
                what, ": q must be [", B, ", ", T, ", heads, ", d, "] of the keys' type and device");
    q_out = at::empty({B, T, q->size(2), d}, q->options());
    a.q_out = q_out.data_ptr();
    if (q_out.numel() == 0) a.q = Rows{};
  }
  if (freq.has_value() && freq->defined()) {
    TORCH_CHECK(freq->device() == ck.device() && freq->scalar_type() == at::kFloat && freq->dim() == 1 &&
                    freq->is_contiguous() && 2 * freq->numel() <= d,
                what, ": inv_freq must be contiguous fp32 of at most head_dim / 2 on the cache's device");
    a.freq = freq->data_ptr<float>();
    a.n = (int)freq->numel();
  }
  a.amplitude = (float)amplitude;
  a.half = half;
  a.offset = offset;
  a.T = (int)T;
  a.S = (int)ck.size(2);
  a.d = (int)d;
  if (B == 0 || T == 0) return q_out;
  const int kind = cache_kind(ck.scalar_type(), what);
  TB_DISPATCH_FLOAT(k.scalar_type(), what, [&] {
    TB_DISPATCH_CACHE(kind, what, [&] { launch_write<scalar_t, cache_t>(a, B); });
  });
  check_launch(what);
  return q_out;
}

std::vector<at::Tensor> kv_cache_read(const at::Tensor& ck, const at::Tensor& cv,
                                      const c10::optional<at::Tensor>& ks, const c10::optional<at::Tensor>& vs,
                                      const at::Tensor& lengths, int64_t n, at::ScalarType dtype) {
  const char* what = "kv_cache_read";
  ReadArgs a{};
  a.ck = cache_view(ck, ks, what);
  a.cv = cache_view(cv, vs, what);
  TORCH_CHECK(ck.sizes() == cv.sizes() && ck.scalar_type() == cv.scalar_type() && ck.device() == cv.device(), what,
              ": the key and value caches must have one shape, type and device");
  const int64_t B = ck.size(0), H = ck.size(1), S = ck.size(2), d = ck.size(3);
  TORCH_CHECK(lengths.device() == ck.device() && lengths.scalar_type() == at::kLong && lengths.dim() == 1 &&
                  lengths.size(0) == B, what, ": lengths must be int64 [", B, "] on the cache's device");
  TORCH_CHECK(n >= 0 && n <= S, what, ": at most the cache's ", S, " slots can be read");
  TORCH_CHECK(B * H < 65536, what, ": at most 65535 (sequence, head) pairs in one call");
  const at::cuda::CUDAGuard g(ck.device());
  at::Tensor ko = at::empty({B, H, n, d}, ck.options().dtype(dtype)), vo = at::empty_like(ko);
  if (ko.numel() == 0) return {ko, vo};
  a.ko = ko.data_ptr();
  a.vo = vo.data_ptr();
  a.lengths = lengths.data_ptr<int64_t>();
  a.len_s = lengths.stride(0);
  a.H = (int)H;
  a.S = (int)S;
  a.n = (int)n;
  a.d = (int)d;
  const int64_t vecs = n * (d / 8);
  const dim3 grid((unsigned)((vecs + kThreads - 1) / kThreads), (unsigned)(B * H), 2);
  const int kind = cache_kind(ck.scalar_type(), what);
  TB_DISPATCH_FLOAT(dtype, what, [&] {
    TB_DISPATCH_CACHE(kind, what,
                      [&] { kv_read_kernel<cache_t, scalar_t><<<grid, kThreads, 0, stream()>>>(a); });
  });
  check_launch(what);
  return {ko, vo};
}

}  // namespace tb
