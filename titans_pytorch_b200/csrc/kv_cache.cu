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
// Each new row is read once (a half-layout row finds its partner elements in
// L1) and written once.  4 prompts of up to 4096 tokens, 16 heads of 96, fp8:
// the write takes 110 us, bound by its instructions (rotation, two divisions and
// eight conversions a lane; memory alone would take 30), the read of 8192 slots
// 50 us, 75 % of the copy rate.
#include <ATen/MemoryOverlap.h>

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
  int tokens;  // of a block
  FastDiv by_token;  // rows of a token
  float amplitude;
  int half;
};

// 8 elements of row x from column c, rotated.  cs, sn: the token's tables,
// padded with (1, 0) to a multiple of 8 pairs.
template <typename T>
__device__ __forceinline__ void rotated8(const T* x, int c, const float* cs, const float* sn, int n, bool half, float (&v)[8]) {
  load8<T>(x + c, v);
  if (c >= 2 * n) return;
  if (!half) {
    float a[4], b[4];
    table_load(cs + c / 2, a);
    table_load(sn + c / 2, b);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (c + i >= 2 * n) break;  // not times (1, 0): an infinity would spoil the other of its pair
      const float p = v[i], q = v[i + 1];
      v[i] = p * a[i / 2] - q * b[i / 2];
      v[i + 1] = p * b[i / 2] + q * a[i / 2];
    }
  } else if (n % 8 == 0) {  // the partners are a vector of their own
    const bool low = c < n;
    const int at = low ? c : c - n;
    float w[8], a[8], b[8];
    load8<T>(x + (low ? c + n : c - n), w);
    table_load(cs + at, a);
    table_load(sn + at, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = low ? v[i] * a[i] - w[i] * b[i] : w[i] * b[i] + v[i] * a[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = c + i;
      if (j < n)
        v[i] = v[i] * cs[j] - to_f<T>(x[j + n]) * sn[j];
      else if (j < 2 * n)
        v[i] = to_f<T>(x[j - n]) * sn[j - n] + v[i] * cs[j - n];
    }
  }
}

// Block = a few tokens of one sequence, all their heads: first the tokens' cos /
// sin, then LANES lanes per row (a power of two >= d / 8), 8 elements a lane.
template <typename T, typename C, int LANES>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(WriteArgs a) {
  extern __shared__ __align__(16) float tab[];  // [token] cos, then sin of the pairs
  const int np = (a.n + 7) & ~7;
  const int t0 = blockIdx.x * a.tokens, b = blockIdx.y;
  const int toks = min(a.tokens, a.T - t0);
  const int64_t start = a.start[b * a.start_s];
  int64_t count = a.count ? a.count[b * a.count_s] : a.T;
  count = min(max(count, (int64_t)0), (int64_t)a.T);
  // a token that a later one of this call would overwrite is not stored, nor one before position 0
  auto stored = [&](int t) { return t < count && t >= count - a.S && start + t >= 0; };
  for (int i = threadIdx.x; i < toks * np; i += kThreads) {
    const int k = i / np, p = i - k * np;
    const float2 cs = p < a.n ? rope_cos_sin(start + t0 + k + a.offset, a.freq[p], a.amplitude) : make_float2(1.f, 0.f);
    tab[2 * k * np + p] = cs.x;
    tab[(2 * k + 1) * np + p] = cs.y;
  }
  __shared__ int sh_slot;  // of the block's first token (where it has one): one 64-bit division a block
  if (threadIdx.x == 0) sh_slot = (int)((start + t0) % a.S);
  __syncthreads();
  const int lane = threadIdx.x % LANES;
  const int c = lane * 8;
  const bool on = c < a.d;
  const int per_tok = a.q.H + a.k.H + a.v.H, rows = toks * per_tok;
  // whole warps stay in the loop for the shuffles
  for (int r0 = 0; r0 < rows; r0 += kThreads / LANES) {
    const int row = r0 + threadIdx.x / LANES;
    int r;
    const int k = a.by_token(row, r), t = t0 + k;
    const float* cs = tab + 2 * k * np;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row < rows && r < a.q.H && on) {
      const T* src = (const T*)a.q.p + b * a.q.sb + t * a.q.st + r * a.q.sh;
      rotated8<T>(src, c, cs, cs + np, a.n, a.half, x);
      store8<T>((T*)a.q_out + (((int64_t)b * a.T + t) * a.q.H + r) * a.d + c, x);
    }
    const int kv = r - a.q.H;
    const bool mine = row < rows && kv >= 0 && stored(t);
    const bool is_v = kv >= a.k.H;
    const int h = is_v ? kv - a.k.H : kv;
    if (mine && on) {
      const Rows& in = is_v ? a.v : a.k;
      const T* src = (const T*)in.p + b * in.sb + t * in.st + h * in.sh;
      if (is_v)
        load8<T>(src + c, x);
      else
        rotated8<T>(src, c, cs, cs + np, a.n, a.half, x);
    }
    // (positions of a block that begins before position 0 wrap here, not in C++'s remainder)
    int64_t slot = sh_slot + k;
    slot = slot < 0 ? slot + a.S : slot;
    if (slot >= a.S) slot %= a.S;
    const CacheView& dst = is_v ? a.cv : a.ck;
    if (!__any_sync(0xffffffffu, mine)) continue;  // queries only
    if constexpr (CacheTraits<C>::scaled) {
      // the largest magnitude by its bits: infinities and NaN come out above every number
      uint32_t top_bits = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) top_bits = max(top_bits, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) top_bits = max(top_bits, __shfl_xor_sync(0xffffffffu, top_bits, o));
      const float amax = __uint_as_float(top_bits);
      constexpr float top = CacheTraits<C>::top;
      const bool bad = top_bits >= 0x7f800000u;
      const bool full = amax >= 7.888609052210118e-31f && !bad;  // 2^-100
      const float inv = full ? top / amax : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = bad ? 0.f : x[i] * inv;
      if (mine && lane == 0)
        dst.scale[b * dst.qb + h * dst.qh + slot * dst.qs] = bad ? __int_as_float(0x7fffffff) : full ? amax / top : 1.f;
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
  FastDiv by_row;  // pieces of a row
};

// Row i of the output: the i-th of the newest min(length, slots, n) tokens, in
// order; zeros behind the last.  Block = rows_per_block rows of one (sequence,
// head, keys or values); one thread moves four times 8 elements.
template <typename C, typename T>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(ReadArgs a) {
  const int h = blockIdx.y % a.H, b = blockIdx.y / a.H;
  const bool is_v = blockIdx.z;
  const CacheView& src = is_v ? a.cv : a.ck;
  const int64_t len = max(a.lengths[b * a.len_s], (int64_t)0);
  const int held = (int)min(len, (int64_t)min(a.S, a.n));
  __shared__ int sh_first;  // the first token's slot: one 64-bit division a block
  if (threadIdx.x == 0) sh_first = (int)((len - held) % a.S);
  __syncthreads();
  // four rows' pieces in flight a thread
  constexpr int U = 4;
  float x[U][8];
  int at[U], col[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    int c;
    const int i = a.by_row((int)((blockIdx.x * U + u) * kThreads + threadIdx.x), c);
    c *= 8;
    at[u] = i;
    col[u] = c;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[u][k] = 0.f;
    if (i < held) {
      int64_t slot = sh_first + i;
      if (slot >= a.S) slot -= a.S;
      load8<C>((const C*)src.data + b * src.sb + h * src.sh + slot * src.ss + c, x[u]);
      if constexpr (CacheTraits<C>::scaled) {
        const float s = src.scale[b * src.qb + h * src.qh + slot * src.qs];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[u][k] *= s;
      }
    }
  }
  T* dst = (T*)(is_v ? a.vo : a.ko);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (at[u] < a.n) store8<T>(dst + ((int64_t)blockIdx.y * a.n + at[u]) * a.d + col[u], x[u]);
}

// `hold` keeps the copy that unaligned rows need, and rows of the cache itself, which the call overwrites.
Rows rows_of(const at::Tensor& x, at::Tensor& hold, const at::Tensor& ck, const at::Tensor& cv, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 4, what, ": new tokens must be CUDA tensors [B, T, H, d]");
  const at::cuda::CUDAGuard g(x.device());
  const int64_t size = x.element_size();
  const bool fits = x.stride(3) == 1 && x.stride(0) * size % 16 == 0 && x.stride(1) * size % 16 == 0 &&
                    x.stride(2) * size % 16 == 0 && aligned16(x);
  if (x.is_alias_of(ck) || x.is_alias_of(cv))
    hold = x.clone(at::MemoryFormat::Contiguous);
  else
    hold = fits ? x : contig16(x);
  return Rows{hold.data_ptr(), hold.stride(0), hold.stride(1), hold.stride(2), (int)hold.size(2)};
}

// Blocks write rows in any order: no two rows may be the same memory.
void check_distinct(const at::Tensor& a, const at::Tensor& b, const char* what) {
  using at::MemOverlapStatus;
  const MemOverlapStatus both = at::get_overlap_status(a, b);
  TORCH_CHECK(at::has_internal_overlap(a) != at::MemOverlap::Yes && at::has_internal_overlap(b) != at::MemOverlap::Yes &&
                  both != MemOverlapStatus::Full && both != MemOverlapStatus::Partial,
              what, ": a cache whose rows share memory cannot be written");
}

template <typename T, typename C>
void launch_write(WriteArgs a, int64_t B) {
  // several tokens a block, so that the table's latency is paid less often, while the GPU is full without it
  a.tokens = (int)std::max<int64_t>(1, std::min<int64_t>(2, B * a.T / (num_sms() * 4)));
  a.by_token = FastDiv((uint32_t)(a.q.H + a.k.H + a.v.H));
  const dim3 grid((unsigned)((a.T + a.tokens - 1) / a.tokens), (unsigned)B);
  const size_t smem = (size_t)a.tokens * ((a.n + 7) & ~7) * 2 * sizeof(float);
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
  check_distinct(ck, cv, what);
  if (a.ck.scale) check_distinct(*ks, *vs, what);
  at::Tensor hold_k, hold_v, hold_q;
  a.k = rows_of(k, hold_k, ck, cv, what);
  a.v = rows_of(v, hold_v, ck, cv, what);
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
    a.q = rows_of(*q, hold_q, ck, cv, what);
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
  if (B == 0 || T == 0 || a.q.H + 2 * H == 0) return q_out;
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
  a.by_row = FastDiv((uint32_t)(d / 8));
  const int64_t vecs = n * (d / 8);
  TORCH_CHECK(vecs < (1ll << 31) - 8 * kThreads, what, ": too many slots in one call");
  const dim3 grid((unsigned)((vecs + 4 * kThreads - 1) / (4 * kThreads)), (unsigned)(B * H), 2);
  const int kind = cache_kind(ck.scalar_type(), what);
  TB_DISPATCH_FLOAT(dtype, what, [&] {
    TB_DISPATCH_CACHE(kind, what,
                      [&] { kv_read_kernel<cache_t, scalar_t><<<grid, kThreads, 0, stream()>>>(a); });
  });
  check_launch(what);
  return {ko, vo};
}

}  // namespace tb
