// Attention of one query token per sequence over a key/value cache and, in
// front of it, a prefix that every sequence of the batch shares.
//
//   s_j = scale * q . k_j,  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),
//   lse = m + log sum_j exp(s_j - m),  j over prefix keys and cache slots.
//
// A softmax over a union of key sets is the weighted sum of the softmaxes over
// each set: a piece of the keys gives (m, l, O) with O = sum exp2(s - m) v and
// l = sum exp2(s - m), and pieces are joined by rescaling to the larger m.  So
// the keys of a row are split over blocks, every block leaves (m, l, O) in fp32
// in a workspace, and a second kernel joins them in a fixed order.  A row with
// no key at all gives zeros and lse = -inf.
#include "kv_cache.cuh"

namespace tb {
namespace {

// Keys of one kind (the cache, or the shared prefix) seen by kernel.
struct KeySource {
  CacheView k, v;
  const int64_t* lengths;  // per sequence, or null: `fixed` keys
  int64_t len_s;
  int64_t fixed;
  int S;        // ring size
  int window;   // newest keys visible
};

struct DecodeArgs {
  KeySource src;
  const void* q;
  int q_type;
  int64_t sqb, sqh;
  float* part;        // [rows][splits][d + 2]: O, m, l
  int splits, split0; // pieces a row has in all; the first of this launch
  int nsplit;         // pieces of this launch
  int B, Hq, Hkv, group, d;
  float scale_log2;
};

__device__ __forceinline__ float load_q(const void* q, int type, int64_t i) {
  if (type == KV_F32) return ((const float*)q)[i];
  if (type == KV_BF16) return to_f<__nv_bfloat16>(((const __nv_bfloat16*)q)[i]);
  return to_f<__half>(((const __half*)q)[i]);
}

// First visible slot and number of visible keys of sequence b.
__device__ __forceinline__ void visible(const KeySource& s, int b, int& first, int& count) {
  if (s.lengths == nullptr) {
    first = 0;
    count = (int)s.fixed;
    return;
  }
  const int64_t len = max(s.lengths[b * s.len_s], (int64_t)0);
  const int64_t n = min(min(len, (int64_t)s.S), (int64_t)s.window);
  count = (int)n;
  // all slots of a full ring, in any order: start at 0
  first = n == s.S ? 0 : (int)((len - n) % s.S);
}

template <typename C> struct Raw8 {
  static constexpr int W = sizeof(C) * 8 / 4;
  uint32_t w[W];
  __device__ __forceinline__ void load(const C* p) {
    if constexpr (W == 2) {
      const uint2 a = *reinterpret_cast<const uint2*>(p);
      w[0] = a.x; w[1] = a.y;
    } else {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const uint4 a = reinterpret_cast<const uint4*>(p)[i / 4];
        w[i] = a.x; w[i + 1] = a.y; w[i + 2] = a.z; w[i + 3] = a.w;
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void unpack(float (&v)[8]) const {
    const C* c = reinterpret_cast<const C*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f<C>(c[i]);
  }
};

constexpr int kWarps = 4, kThreads = 32 * kWarps;

// fp32 arithmetic on the CUDA cores, any head dimension (a multiple of 8 up to
// 256), any cache type.  LANES lanes share a key, 8 elements each; every group
// of lanes keeps its own running (m, l, O) for G query heads of one key head.
template <typename C, int LANES, int G>
__global__ void __launch_bounds__(kThreads) decode_simt_kernel(DecodeArgs a) {
  constexpr int KPW = 32 / LANES, GROUPS = KPW * kWarps, U = 4;
  __shared__ float sm_o[GROUPS][G][LANES * 8];
  __shared__ float sm_m[GROUPS][G], sm_l[GROUPS][G];
  const int split = blockIdx.x % a.nsplit, gt = blockIdx.x / a.nsplit;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / LANES, c = (lane % LANES) * 8;
  const bool on = c < a.d;
  const int g0 = gt * G;
  float q[G][8], o[G][8], m[G], l[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o[g][e] = 0.f;
      q[g][e] = on && g0 + g < a.group
                    ? load_q(a.q, a.q_type, b * a.sqb + (int64_t)(hk * a.group + g0 + g) * a.sqh + c + e) * a.scale_log2
                    : 0.f;
    }
  }
  int first, count;
  visible(a.src, b, first, count);
  const int per = (count + a.nsplit - 1) / a.nsplit;
  const int lo = min(split * per, count), hi = min(lo + per, count);
  const C* kb = (const C*)a.src.k.data + b * a.src.k.sb + hk * a.src.k.sh + c;
  const C* vb = (const C*)a.src.v.data + b * a.src.v.sb + hk * a.src.v.sh + c;
  for (int base = lo + warp * U * KPW; base < hi; base += kWarps * U * KPW) {
    Raw8<C> kr[U], vr[U];
    float ks[U], vs[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + u * KPW + sub;
      ok[u] = i < hi;
      int slot = first + i;
      if (slot >= a.src.S) slot -= a.src.S;
      ks[u] = vs[u] = 1.f;
      if (ok[u] && on) {
        kr[u].load(kb + slot * a.src.k.ss);
        vr[u].load(vb + slot * a.src.v.ss);
      } else {  // masked keys never enter the arithmetic: their slots may hold anything
        kr[u].zero();
        vr[u].zero();
      }
      if constexpr (CacheTraits<C>::scaled) {
        if (ok[u]) {
          ks[u] = a.src.k.scale[b * a.src.k.qb + hk * a.src.k.qh + slot * a.src.k.qs];
          vs[u] = a.src.v.scale[b * a.src.v.qb + hk * a.src.v.qh + slot * a.src.v.qs];
        }
      }
    }
    float s[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float k[8];
      kr[u].unpack(k);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) t = fmaf(q[g][e], k[e], t);
        s[u][g] = t;
      }
    }
#pragma unroll
    for (int x = LANES / 2; x > 0; x >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int g = 0; g < G; ++g) s[u][g] += __shfl_xor_sync(0xffffffffu, s[u][g], x);
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) vr[u].unpack(v[u]);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float mx = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u][g] = ok[u] ? s[u][g] * ks[u] : -INFINITY;
        mx = fmaxf(mx, s[u][g]);
      }
      const float use = mx == -INFINITY ? 0.f : mx;
      const float corr = exp2f(m[g] - use);
      m[g] = mx;
      l[g] *= corr;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[g][e] *= corr;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = exp2f(s[u][g] - use);
        l[g] += p;
        const float pv = ok[u] ? p * vs[u] : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[g][e] = fmaf(pv, v[u][e], o[g][e]);
      }
    }
  }
  const int grp = warp * KPW + sub;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (lane % LANES == 0) {
      sm_m[grp][g] = m[g];
      sm_l[grp][g] = l[g];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sm_o[grp][g][c + e] = o[g][e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * a.d; i += kThreads) {
    const int g = i / a.d, e = i - g * a.d;
    if (g0 + g >= a.group) continue;
    float mx = -INFINITY;
    for (int x = 0; x < GROUPS; ++x) mx = fmaxf(mx, sm_m[x][g]);
    const float use = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, den = 0.f;
    for (int x = 0; x < GROUPS; ++x) {
      const float w = exp2f(sm_m[x][g] - use);
      sum += w * sm_o[x][g][e];
      den += w * sm_l[x][g];
    }
    const int64_t row = (int64_t)b * a.Hq + hk * a.group + g0 + g;
    float* dst = a.part + (row * a.splits + a.split0 + split) * (a.d + 2);
    dst[e] = sum;
    if (e == 0) {
      dst[a.d] = mx;
      dst[a.d + 1] = den;
    }
  }
}

// Joins the pieces of each row: one warp a row, split order.
template <typename T>
__global__ void __launch_bounds__(kThreads) decode_join_kernel(const float* __restrict__ part, int splits, int d,
                                                               int64_t rows, T* __restrict__ out,
                                                               float* __restrict__ lse) {
  const int64_t row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  const float* p = part + row * splits * (d + 2);
  float m = -INFINITY;
  for (int s = lane; s < splits; s += 32) m = fmaxf(m, p[(int64_t)s * (d + 2) + d]);
  m = warp_max(m);
  const float use = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float* ps = p + (int64_t)s * (d + 2);
    l += exp2f(ps[d] - use) * ps[d + 1];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int e = lane; e < d; e += 32) {
    float o = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float* ps = p + (int64_t)s * (d + 2);
      o += exp2f(ps[d] - use) * ps[e];
    }
    out[row * d + e] = from_f<T>(o * inv);
  }
  if (lse && lane == 0) lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <typename C, int LANES>
void launch_simt(const DecodeArgs& a) {
  const int G = a.group == 1 ? 1 : 4;
  const dim3 grid((unsigned)(a.nsplit * ((a.group + G - 1) / G)), (unsigned)a.Hkv, (unsigned)a.B);
  if (G == 1)
    decode_simt_kernel<C, LANES, 1><<<grid, kThreads, 0, stream()>>>(a);
  else
    decode_simt_kernel<C, LANES, 4><<<grid, kThreads, 0, stream()>>>(a);
}

void launch_source(const DecodeArgs& a, int kind) {
  TB_DISPATCH_CACHE(kind, "decode_attention", [&] {
    if (a.d <= 64)
      launch_simt<cache_t, 8>(a);
    else if (a.d <= 128)
      launch_simt<cache_t, 16>(a);
    else
      launch_simt<cache_t, 32>(a);
  });
}

// Pieces for `keys` keys a row: enough blocks for two rounds of the GPU, no
// piece shorter than 128 keys.
int pieces(int64_t keys, int64_t blocks) {
  const int64_t want = (2 * 4 * num_sms() + blocks - 1) / blocks;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, (keys + 127) / 128, 64}));
}

// The prefix [P, Hkv, d] as a key source; `hold` keeps the copy that unaligned rows need.
CacheView prefix_view(const at::Tensor& p, at::Tensor& hold) {
  const int64_t size = p.element_size();
  const bool fits = p.stride(2) == 1 && p.stride(0) * size % 16 == 0 && p.stride(1) * size % 16 == 0 && aligned16(p);
  hold = fits ? p : contig16(p);
  return CacheView{hold.data_ptr(), nullptr, 0, hold.stride(1), hold.stride(0), 0, 0, 0};
}

}  // namespace

std::vector<at::Tensor> decode_attention(const at::Tensor& q, const at::Tensor& ck, const at::Tensor& cv,
                                         const c10::optional<at::Tensor>& ks, const c10::optional<at::Tensor>& vs,
                                         const at::Tensor& lengths, const c10::optional<at::Tensor>& pk,
                                         const c10::optional<at::Tensor>& pv, int64_t window, double scale,
                                         bool want_lse) {
  const char* what = "decode_attention";
  TORCH_CHECK(q.is_cuda() && q.dim() == 3, what, ": q must be a CUDA tensor [B, heads, d]");
  TORCH_CHECK(q.scalar_type() == at::kFloat || q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, what,
              ": q must be float32, bfloat16 or float16");
  DecodeArgs a{};
  a.src.k = cache_view(ck, ks, what);
  a.src.v = cache_view(cv, vs, what);
  const int64_t B = q.size(0), Hq = q.size(1), d = q.size(2), Hkv = ck.size(1), S = ck.size(2);
  TORCH_CHECK(ck.sizes() == cv.sizes() && ck.scalar_type() == cv.scalar_type() && ck.device() == cv.device(), what,
              ": the key and value caches must have one shape, type and device");
  TORCH_CHECK(ck.device() == q.device() && ck.size(0) == B && ck.size(3) == d, what, ": the cache must be [", B,
              ", heads, slots, ", d, "] on the queries' device");
  TORCH_CHECK(Hkv >= 1 && Hq % Hkv == 0, what, ": ", Hq, " query heads are not a multiple of ", Hkv, " key heads");
  TORCH_CHECK(lengths.device() == q.device() && lengths.scalar_type() == at::kLong && lengths.dim() == 1 &&
                  lengths.size(0) == B, what, ": lengths must be int64 [", B, "] on the queries' device");
  TORCH_CHECK(window >= 1, what, ": the window must hold at least one key");
  TORCH_CHECK(q.stride(2) == 1 || d == 1, what, ": q rows must be contiguous");
  TORCH_CHECK(B < 65536 && Hkv < 65536, what, ": at most 65535 sequences and key heads in one call");
  at::Tensor hold_pk, hold_pv;
  const bool has_prefix = pk.has_value() && pk->defined() && pk->size(0) > 0;
  int64_t P = 0;
  if (has_prefix) {
    TORCH_CHECK(pv.has_value() && pv->defined(), what, ": prefix keys come with prefix values");
    P = pk->size(0);
    for (const at::Tensor* t : {&*pk, &*pv})
      TORCH_CHECK(t->device() == q.device() && t->scalar_type() == q.scalar_type() && t->dim() == 3 &&
                      t->size(0) == P && t->size(1) == Hkv && t->size(2) == d && P < (1ll << 30),
                  what, ": the prefix must be [P, ", Hkv, ", ", d, "] of the queries' type and device");
  }
  const at::cuda::CUDAGuard g(q.device());
  at::Tensor out = at::empty({B, Hq, d}, q.options());
  at::Tensor lse = want_lse ? at::empty({B, Hq}, q.options().dtype(at::kFloat)) : at::Tensor();
  if (out.numel() == 0) return {out, lse};
  a.src.lengths = lengths.data_ptr<int64_t>();
  a.src.len_s = lengths.stride(0);
  a.src.S = (int)S;
  a.src.window = (int)std::min<int64_t>(window, 1ll << 30);
  a.q = q.data_ptr();
  a.q_type = cache_kind(q.scalar_type(), what);
  a.sqb = q.stride(0);
  a.sqh = q.stride(1);
  a.B = (int)B;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.group = (int)(Hq / Hkv);
  a.d = (int)d;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  const int64_t blocks = B * Hkv;
  const int cs = pieces(std::min<int64_t>(S, window), blocks);
  const int ps = has_prefix ? pieces(P, blocks) : 0;
  a.splits = cs + ps;
  at::Tensor part = at::empty({B * Hq, a.splits, d + 2}, q.options().dtype(at::kFloat));
  a.part = part.data_ptr<float>();
  if (has_prefix) {
    DecodeArgs p = a;
    p.src.k = prefix_view(*pk, hold_pk);
    p.src.v = prefix_view(*pv, hold_pv);
    p.src.lengths = nullptr;
    p.src.fixed = P;
    p.src.S = 1 << 30;
    p.nsplit = ps;
    p.split0 = 0;
    launch_source(p, a.q_type);
    check_launch(what);
  }
  a.nsplit = cs;
  a.split0 = ps;
  launch_source(a, cache_kind(ck.scalar_type(), what));
  check_launch(what);
  const int64_t rows = B * Hq;
  TB_DISPATCH_FLOAT(q.scalar_type(), what, [&] {
    decode_join_kernel<scalar_t><<<(unsigned)((rows + kWarps - 1) / kWarps), kThreads, 0, stream()>>>(
        a.part, a.splits, (int)d, rows, (scalar_t*)out.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr);
  });
  check_launch(what);
  return {out, lse};
}

}  // namespace tb
