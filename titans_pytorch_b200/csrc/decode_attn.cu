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
  bool early;         // may start while the launch in front of it (the prefix) runs
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

// Launches of one call overlap: a kernel launched with `early` may start while
// the one in front of it still runs, and waits for its results where it says so.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }

template <typename... P, typename... A>
void launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, bool early, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 1 : 0;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
}

// fp32 arithmetic on the CUDA cores, any head dimension (a multiple of 8 up to
// 256), any cache type.  LANES lanes share a key, 8 elements each; every group
// of lanes keeps its own running (m, l, O) for G query heads of one key head.
template <typename C, int LANES, int G>
__global__ void __launch_bounds__(kThreads) decode_simt_kernel(DecodeArgs a) {
  constexpr int KPW = 32 / LANES, GROUPS = KPW * kWarps, U = 4;
  __shared__ float sm_o[GROUPS][G][LANES * 8];
  __shared__ float sm_m[GROUPS][G], sm_l[GROUPS][G];
  let_next_start();
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
  // the kernel behind this one waits for this one alone: so this one ends after the one in front of it
  wait_for_previous();
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

// Joins the pieces of each row, in a fixed order: one block a row, warp w takes
// pieces w, w + 8, ... (one warp walking all pieces took 0.5 us a piece).
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) decode_join_kernel(const float* __restrict__ part, int splits, int d,
                                                                      T* __restrict__ out, float* __restrict__ lse) {
  __shared__ float sm_o[kJoinWarps][256], sm_l[kJoinWarps], sm_m[kJoinWarps];
  const int64_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* p = part + row * splits * (d + 2);
  wait_for_previous();
  float m = -INFINITY;
  for (int s = threadIdx.x; s < splits; s += 32 * kJoinWarps) m = fmaxf(m, p[(int64_t)s * (d + 2) + d]);
  m = warp_max(m);
  if (lane == 0) sm_m[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) m = fmaxf(m, sm_m[w]);
  const float use = m == -INFINITY ? 0.f : m;
  float o[8], l = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = 0.f;
#pragma unroll 4
  for (int s = warp; s < splits; s += kJoinWarps) {
    const float* ps = p + (int64_t)s * (d + 2);
    const float f = exp2f(ps[d] - use);
    l += f * ps[d + 1];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (lane + 32 * k < d) o[k] += f * ps[lane + 32 * k];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (lane + 32 * k < d) sm_o[warp][lane + 32 * k] = o[k];
  if (lane == 0) sm_l[warp] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) l += sm_l[w];
  const int e = threadIdx.x;
  if (e < d) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) sum += sm_o[w][e];
    out[row * d + e] = from_f<T>(l == 0.f ? 0.f : sum / l);
  }
  if (lse && e == 0) lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// ------------------------------------------------------------- tensor cores
// Queries in bf16 or fp16 over keys of the same type or of 8 bits.
//
// A warp takes 16 keys at a time against 8 * NQ query rows, as S^T = K Q^T and
// O^T += V^T P^T on mma.m16n8k16: keys (then head dimensions) are the 16 rows,
// queries the 8 columns, so a single query wastes little.  The order of the
// contracted index is free, so each lane loads whole 16-byte pieces of its key
// rows straight from memory into operand registers (no shared memory): lane
// (r, c) = (lane / 4, lane % 4) holds keys r and r + 8, pieces c of 8 (16 at 8
// bits) dimensions.  For V the lane holds the four keys 2c, 2c+1, 2c+8, 2c+9 and
// piece r; byte permutes pair up neighbouring keys.  P passes from the score
// layout to the operand layout by an 8x8 transpose in registers.
//
// Bound by memory: decoding reads every key once for a handful of queries, far
// below the tensor cores' rate even at mma.sync's, so tcgen05 with its 128-row
// tiles would gain nothing.  K registers are reloaded as soon as the scores have
// read them, V registers after the product, so each warp keeps 4 to 8 KB in
// flight.
//
// The running maximum m moves only when a score exceeds it by more than 8 (in
// log2), so most steps need no exchange between lanes.  Weights are rounded to 16
// bits for the product (half a step each); sums of them are taken before that, in
// fp32.  fp16 weights are aimed at 2^7 (exp2(s - m + 7), at most 2^15): what
// counts 2^-21 of the largest still has all its bits.
//
// 8-bit keys and values are exact in fp16; a value's scale is multiplied into its
// weight before that is rounded.  So m follows score + log2(value scale) there.
// The scale of a row says how large its values are, except where they are all
// zero (the scale is 1 then, far above that of small values), or where it is no
// positive number.  Such rows count with kNoLift instead: they move m only as
// far as keeps their weight, and the sum of 2^20 such, within fp32, and take
// precision only from what weighs less than 2^-111 of them.  Which rows are zero
// is looked up in the values only where one of them would move m (64 ragged int8
// sequences of 12 heads, up to 8192 keys: 131 us; with the scale taken as it is 129).

template <typename T> struct Pair;  // two packed 16-bit floats
template <> struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <> struct Pair<__half> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
// log2 of the value scale that rows without magnitude count with
constexpr float kNoLift = -90.f;
// log2 of what the largest weight is aimed at
template <typename TM> constexpr float kAim = std::is_same<TM, __half>::value ? 7.f : 0.f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// 8-bit numbers widened to fp16, exactly.  The ALU pipe is what limits the 8-bit
// kinds (half the issue rate), so these are counted in its operations.
template <typename C> struct Widen;
template <> struct Widen<int8_t> {
  // bytes 0 and 2 of p: 1024 + (b + 128) less 1152
  static __device__ __forceinline__ uint32_t even(uint32_t p) {
    const uint32_t x = (p & 0x00ff00ffu) ^ 0x64806480u, y = 0x64806480u;
    __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  // a key's four bytes as two pairs: (0, 2) and (1, 3)
  static __device__ __forceinline__ void key(uint32_t w, uint32_t& a, uint32_t& b) {
    a = even(w);
    b = even(w >> 8);
  }
  // byte e of two values
  static __device__ __forceinline__ uint32_t values(uint32_t v0, uint32_t v1, int e) {
    return even(__byte_perm(v0, v1, e | ((4 + e) << 8)));
  }
};
template <> struct Widen<e4m3> {
  static __device__ __forceinline__ uint32_t two(uint32_t p) {  // bytes 0 and 1
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(p & 0xffffu), __NV_E4M3);
    return (uint32_t)r.x | ((uint32_t)r.y << 16);
  }
  static __device__ __forceinline__ void key(uint32_t w, uint32_t& a, uint32_t& b) {  // pairs (0, 1) and (2, 3)
    a = two(w);
    b = two(w >> 16);
  }
  static __device__ __forceinline__ uint32_t values(uint32_t v0, uint32_t v1, int e) {
    return two(__byte_perm(v0, v1, e | ((4 + e) << 4)));
  }
};

template <typename C, int D> struct Layout {
  static constexpr bool k16 = sizeof(C) == 2;
  static constexpr int CK = k16 ? 8 : D % 64 == 0 ? 16 : 8;             // dimensions in a lane's piece of a key
  static constexpr int CV = k16 ? (D % 64 == 0 ? 8 : 4) : D == 128 ? 16 : D == 64 ? 8 : 4;  // of a value
  static constexpr int KW = D / 4 * sizeof(C) / 4;                     // words of a key a lane holds
  static constexpr int VW = D / 8 * sizeof(C) / 4;                     // words of a value (may end mid-word at D = 96)
  // the dimension, of the four of a step, that is element y of pair x
  static __device__ __forceinline__ int at(int x, int y) {
    return std::is_same<C, int8_t>::value ? x + 2 * y : 2 * x + y;
  }
  static constexpr int U = D == 64 ? (k16 ? 2 : 4) : k16 ? 1 : 2;       // groups of 16 keys a step
};

template <int BYTES> __device__ __forceinline__ void load_words(const void* p, uint32_t* w) {
  if constexpr (BYTES == 16) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  } else if constexpr (BYTES == 8) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    w[0] = a.x; w[1] = a.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

struct MmaArgs {
  KeySource cache;
  KeySource ahead;  // a short prefix, which the first piece sees in front of its cache keys (fixed = 0: none)
  bool early;
  const void* q;
  int64_t sqb, sqh;
  float* part;
  void* out;       // written directly when a row has one piece in all
  float* lse;
  int splits, split0, nsplit;
  int piece;                   // keys of a piece
  int Hq, group, rows, tiles;  // query rows of a key head in this launch; tiles of them
  bool shared;                 // rows run over the whole batch (prefix alone)
  float scale_log2;
};

// TM: the type of the products, fp16 beside 8-bit keys, else the queries'.
template <typename TM, int D, int NQ>
struct Warp {
  static constexpr int STEPS = D / 16, R = 8 * NQ;
  uint32_t q[NQ][STEPS][2];
  float o[NQ][STEPS][4];  // [dimension tile][d r / r + 8, query 2c / 2c + 1]
  float m[NQ][2], l[NQ][2], scale[NQ][2];
  int r, c;

  // One kind of keys [lo, hi), every stride-th block of 16 U starting at `block`.
  // PLAIN: rows (and scales) one after the other and no wrap in the range, so
  // that a whole step's addresses are constants away from two pointers.
  template <typename C, bool PLAIN>
  __device__ __forceinline__ void run(const KeySource& s, int b, int hk, int first, int lo, int hi, int block, int stride) {
    using L = Layout<C, D>;
    constexpr bool k8 = CacheTraits<C>::scaled;
    constexpr int U = NQ == 1 ? L::U : 1, KEYS = 16 * U;
    constexpr int NK = L::KW * 4 / (L::CK * (int)sizeof(C)), NV = D / (8 * L::CV);  // pieces
    constexpr int KB = L::CK * sizeof(C), VB = L::CV * sizeof(C), VWP = VB / 4;
    const C* kb = (const C*)s.k.data + b * s.k.sb + hk * s.k.sh + c * L::CK;
    const C* vb = (const C*)s.v.data + b * s.v.sb + hk * s.v.sh + r * L::CV;
    const float* ksb = k8 ? s.k.scale + b * s.k.qb + hk * s.k.qh : nullptr;
    const float* vsb = k8 ? s.v.scale + b * s.v.qb + hk * s.v.qh : nullptr;
    uint32_t kw[U][2][L::KW], vw[U][4][NV * VWP];
    float ks[U][2], vs[U][2];
    auto slot_of = [&](int i) -> int64_t {
      const int x = first + i;
      return x >= s.S ? x - s.S : x;
    };
    auto load_k = [&](int base, bool whole) {
      if (PLAIN && whole) {
        const C* p = kb + (int64_t)(first + base + r) * D;
        const float* ps = k8 ? ksb + first + base + r : nullptr;
        const float* pv = k8 ? vsb + first + base + r : nullptr;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < NK; ++j) load_words<KB>(p + (16 * u + 8 * h) * D + j * 4 * L::CK, &kw[u][h][j * (KB / 4)]);
            if constexpr (k8) {
              ks[u][h] = ps[16 * u + 8 * h];
              vs[u][h] = pv[16 * u + 8 * h];
            }
          }
        return;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = base + 16 * u + 8 * h + r;
          if (i < hi) {
            const int64_t slot = slot_of(i);
            const C* p = kb + slot * s.k.ss;
#pragma unroll
            for (int j = 0; j < NK; ++j) load_words<KB>(p + j * 4 * L::CK, &kw[u][h][j * (KB / 4)]);
            if constexpr (k8) {
              ks[u][h] = ksb[slot * s.k.qs];
              vs[u][h] = vsb[slot * s.v.qs];
            }
          } else if constexpr (k8) {
            ks[u][h] = 0.f;
            vs[u][h] = 0.f;
          }
        }
    };
    auto load_v = [&](int base, bool whole) {
      if (PLAIN && whole) {
        const C* p = vb + (int64_t)(first + base + 2 * c) * D;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int j = 0; j < NV; ++j)
              load_words<VB>(p + (16 * u + (x & 1) + 8 * (x >> 1)) * D + j * 8 * L::CV, &vw[u][x][j * VWP]);
        return;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = base + 16 * u + 2 * c + (x & 1) + 8 * (x >> 1);
          if (i < hi) {
            const C* p = vb + slot_of(i) * s.v.ss;
#pragma unroll
            for (int j = 0; j < NV; ++j) load_words<VB>(p + j * 8 * L::CV, &vw[u][x][j * VWP]);
          } else {  // a weight of zero times whatever the slot holds has to be zero
#pragma unroll
            for (int j = 0; j < NV * VWP; ++j) vw[u][x][j] = 0u;
          }
        }
    };
    int base = lo + block * KEYS;
    if (base >= hi) return;
    bool whole = base + KEYS <= hi;
    load_k(base, whole);
    load_v(base, whole);
    while (true) {
      float sc[U][NQ][4];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[u][n][e] = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
          uint32_t f[2][2];  // [key half][pair]
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if constexpr (k8) {
              Widen<C>::key(kw[u][h][t], f[h][0], f[h][1]);
            } else {
              f[h][0] = kw[u][h][2 * t];
              f[h][1] = kw[u][h][2 * t + 1];
            }
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n) Pair<TM>::mma(sc[u][n], f[0][0], f[1][0], f[0][1], f[1][1], q[n][t][0], q[n][t][1]);
        }
      // the 8-bit kinds watch score + log2(value scale), so that the weights times that scale fit fp16
      float vscale[U][2], grow = -INFINITY, lift[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          lift[u][h] = 0.f;
          if constexpr (k8) {
            vscale[u][h] = vs[u][h];
            lift[u][h] = fmaxf(__log2f(fabsf(vs[u][h])), kNoLift);  // (kNoLift where it is NaN)
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float& x = sc[u][n][2 * h + e];
              x *= k8 ? ks[u][h] * scale[n][e] : scale[n][e];
            }
        }
      if (!whole) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (base + 16 * u + 8 * h + r >= hi)
#pragma unroll
              for (int n = 0; n < NQ; ++n) {
                sc[u][n][2 * h] = -INFINITY;
                sc[u][n][2 * h + 1] = -INFINITY;
              }
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = -INFINITY;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) mx = fmaxf(mx, k8 ? sc[u][n][2 * h + e] + lift[u][h] : sc[u][n][2 * h + e]);
          // m = -inf at first: -inf - -inf is NaN and does not count, a finite score does
          grow = fmaxf(grow, mx - m[n][e]);
        }
      const int next = base + stride * KEYS;
      const bool more = next < hi, next_whole = next + KEYS <= hi;
      if (more) load_k(next, next_whole);
      if (__any_sync(0xffffffffu, grow > 8.f)) {
        if constexpr (k8) {  // rows of zeros
          constexpr uint32_t kMagnitude = std::is_same<C, e4m3>::value ? 0x7f7f7f7fu : 0xffffffffu;  // e4m3 has a -0
          uint32_t full = 0u;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t any = 0u;
#pragma unroll
              for (int j = 0; j < NV * VWP; ++j) any |= vw[u][x][j];
              full |= (any & kMagnitude) ? 1u << (4 * u + x) : 0u;
            }
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) full |= __shfl_xor_sync(0xffffffffu, full, x);
          // from the lanes that hold values 2c, 2c + 1, 2c + 8, 2c + 9 to those of scores r, r + 8
          full = __shfl_sync(0xffffffffu, full, r >> 1);
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (!(full >> (4 * u + 2 * h + (r & 1)) & 1u)) {
                lift[u][h] = kNoLift;
                // the weight may not fit fp16 (a scale that is not finite stays: the row is none of zeros then)
                vscale[u][h] = fabsf(vscale[u][h]) < INFINITY ? 0.f : vscale[u][h];
              } else {
                lift[u][h] = fminf(lift[u][h], 127.f);  // an infinite scale leaves the weights their sum
              }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = m[n][e];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int h = 0; h < 2; ++h) mx = fmaxf(mx, k8 ? sc[u][n][2 * h + e] + lift[u][h] : sc[u][n][2 * h + e]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            const float corr = mx == m[n][e] ? 1.f : ex2(m[n][e] - mx);
            m[n][e] = mx;
            l[n][e] *= corr;
#pragma unroll
            for (int t = 0; t < STEPS; ++t) {
              o[n][t][e] *= corr;
              o[n][t][2 + e] *= corr;
            }
          }
      }
      float use[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) use[n][e] = m[n][e] == -INFINITY ? 0.f : m[n][e] - kAim<TM>;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t p[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float w[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              w[e] = ex2(sc[u][n][2 * h + e] - use[n][e]);
              l[n][e] += w[e];
              if constexpr (k8) w[e] *= vscale[u][h];
            }
            p[n][h] = transpose8x8(Pair<TM>::pack(w[0], w[1]));
          }
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
          uint32_t f[2][2];  // [tile half][key pair]
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int nt = 2 * t + h, e = nt % L::CV, j = nt / L::CV;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              if constexpr (k8) {
                const int w = j * VWP + e / 4;
                f[h][y] = Widen<C>::values(vw[u][2 * y][w], vw[u][2 * y + 1][w], e & 3);
              } else {
                const int w = j * VWP + e / 2;
                f[h][y] = __byte_perm(vw[u][2 * y][w], vw[u][2 * y + 1][w], e & 1 ? 0x7632 : 0x5410);
              }
            }
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n) Pair<TM>::mma(o[n][t], f[0][0], f[1][0], f[0][1], f[1][1], p[n][0], p[n][1]);
        }
      }
      if (!more) break;
      load_v(next, next_whole);
      base = next;
      whole = next_whole;
    }
  }
};

template <typename T, typename C, int D, int NQ>
__global__ void __launch_bounds__(kThreads, NQ == 1 ? 3 : 2) decode_mma_kernel(MmaArgs a) {
  using TM = typename std::conditional<CacheTraits<C>::scaled, __half, T>::type;
  using W = Warp<TM, D, NQ>;
  constexpr int R = W::R, STEPS = W::STEPS;
  let_next_start();
  extern __shared__ float sm[];  // [warp][R][D + 2]: O, m, l (row stride odd against bank conflicts of the transposed store)
  constexpr int RS = D + 3;
  const int split = blockIdx.x % a.nsplit, tile = blockIdx.x / a.nsplit;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = tile * R;  // all warps take the same rows and split the keys
  W w;
  w.r = lane >> 2;
  w.c = lane & 3;
  // row -> (sequence, query head)
  auto place = [&](int row, int& bb, int& h) {
    bb = a.shared ? row / a.group : b;
    h = hk * a.group + (a.shared ? row - bb * a.group : row);
  };
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = row0 + 8 * n + w.r;
    int bb = 0, h = 0;
    if (row < a.rows) place(row, bb, h);
    const T* qp = (const T*)a.q + bb * a.sqb + h * a.sqh;
    // in the order of the dimensions that the keys' pieces have
    float qf[STEPS][2][2], top = 0.f;
#pragma unroll
    for (int t = 0; t < STEPS; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          using L = Layout<C, D>;
          constexpr int CK = L::CK;
          const int d = (t / (CK / 4)) * 4 * CK + w.c * CK + (t % (CK / 4)) * 4 + L::at(x, y);
          qf[t][x][y] = row < a.rows ? to_f<T>(qp[d]) : 0.f;
          top = fmaxf(top, fabsf(qf[t][x][y]));
        }
    // beside 8-bit keys: to fp16 by a power of two that brings the row's largest to [1, 2)
    float down = 1.f, up = 1.f;
    if constexpr (CacheTraits<C>::scaled) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = (__float_as_int(top) >> 23) - 127;
      if (e > -127 && e < 127) {  // both powers are normal numbers
        down = __int_as_float((127 - e) << 23);
        up = __int_as_float((127 + e) << 23);
      }
    }
#pragma unroll
    for (int t = 0; t < STEPS; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) w.q[n][t][x] = Pair<TM>::pack(qf[t][x][0] * down, qf[t][x][1] * down);
#pragma unroll
    for (int e = 0; e < 2; ++e)  // row 2c + e of the scores' layout
      w.scale[n][e] = a.scale_log2 * __shfl_sync(0xffffffffu, up, (2 * w.c + e) * 4);
#pragma unroll
    for (int t = 0; t < STEPS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) w.o[n][t][e] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      w.m[n][e] = -INFINITY;
      w.l[n][e] = 0.f;
    }
  }
  int first = 0, count = 0;
  if (a.shared)
    count = (int)a.cache.fixed;
  else
    visible(a.cache, b, first, count);
  const int lo = min(split * a.piece, count), hi = min(lo + a.piece, count);
  if constexpr (!CacheTraits<C>::scaled)
    if (split == 0 && a.ahead.fixed > 0) w.template run<C, false>(a.ahead, 0, hk, 0, 0, (int)a.ahead.fixed, warp, kWarps);
  const KeySource& src = a.cache;
  const bool plain = src.k.ss == D && src.v.ss == D && first + hi <= src.S &&
                     (!CacheTraits<C>::scaled || (src.k.qs == 1 && src.v.qs == 1));
  if (plain)
    w.template run<C, true>(src, a.shared ? 0 : b, hk, first, lo, hi, warp, kWarps);
  else
    w.template run<C, false>(src, a.shared ? 0 : b, hk, first, lo, hi, warp, kWarps);
  // O, m and l of the warp's rows to shared memory; lane (r, c) holds queries 2c, 2c + 1
  float* mine = sm + warp * R * RS;
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = w.l[n][e];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
      float* row = mine + (8 * n + 2 * w.c + e) * RS;
      if (w.r == 0) {
        row[D] = w.m[n][e] - kAim<TM>;
        row[D + 1] = l;
      }
#pragma unroll
      for (int t = 0; t < STEPS; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          constexpr int CV = Layout<C, D>::CV;
          const int nt = 2 * t + h;
          row[(nt / CV) * 8 * CV + w.r * CV + nt % CV] = w.o[n][t][2 * h + e];
        }
    }
  // the kernel behind this one waits for this one alone: so this one ends after the one in front of it
  wait_for_previous();
  __syncthreads();
  // join the warps that split the keys, in their order
  const int rows = min(R, a.rows - row0);
  for (int i = threadIdx.x; i < rows * D; i += kThreads) {
    const int lr = i / D, e = i - lr * D;
    const float* p = sm + lr * RS;
    constexpr int step = R * RS;
    float mx = p[D];
#pragma unroll
    for (int x = 1; x < kWarps; ++x) mx = fmaxf(mx, p[x * step + D]);
    const float use = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, den = 0.f;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      const float f = ex2(p[x * step + D] - use);
      sum += f * p[x * step + e];
      den += f * p[x * step + D + 1];
    }
    int bb, h;
    place(row0 + lr, bb, h);
    const int64_t row = (int64_t)bb * a.Hq + h;
    if (a.splits == 1) {
      ((T*)a.out)[row * D + e] = from_f<T>(den == 0.f ? 0.f : sum / den);
      if (e == 0 && a.lse) a.lse[row] = den == 0.f ? -INFINITY : (mx + log2f(den)) * 0.6931471805599453f;
    } else {
      float* dst = a.part + (row * a.splits + a.split0 + split) * (D + 2);
      dst[e] = sum;
      if (e == 0) {
        dst[D] = mx;
        dst[D + 1] = den;
      }
    }
  }
}

template <typename T, typename C, int D, int NQ>
void launch_mma(const MmaArgs& a, int Hkv, int B) {
  const size_t smem = (size_t)kWarps * 8 * NQ * (D + 3) * sizeof(float);
  if (smem > 48 * 1024)
    C10_CUDA_CHECK(cudaFuncSetAttribute(decode_mma_kernel<T, C, D, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)smem));
  launch(decode_mma_kernel<T, C, D, NQ>, dim3((unsigned)(a.nsplit * a.tiles), (unsigned)Hkv, (unsigned)(a.shared ? 1 : B)),
         kThreads, smem, a.early, a);
}

// The shared prefix against the queries of the whole batch: 64 or 128 rows a
// block (16 or 32 a warp), so that each key is read from memory once per 128
// rows.  Keys and values go through shared memory (cp.async, three tiles of 64
// keys; rows padded by 16 bytes, which leaves ldmatrix free of bank conflicts),
// as four warps share them; the products are as above.  With 128 rows the tensor
// cores have work for about as long as memory; at mma.sync's rate that suffices.
constexpr int kTile = 64, kStages = 3;

__device__ __forceinline__ void ldmatrix4(uint32_t (&f)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&f)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3])
               : "r"(addr));
}

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(kThreads, D == 64 ? 3 : 2) decode_prefix_kernel(MmaArgs a) {
  constexpr int STEPS = D / 16, R = 8 * NQ, ROW = D * 2 + 16, TILE = kTile * ROW;
  let_next_start();
  extern __shared__ __align__(16) uint8_t smem[];  // [stage][K, V][kTile][ROW]
  const uint32_t sbase = (uint32_t)__cvta_generic_to_shared(smem);
  const int split = blockIdx.x % a.nsplit, tile = blockIdx.x / a.nsplit, hk = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int row0 = (tile * kWarps + warp) * R;
  const int lo = split * a.piece, hi = min(lo + a.piece, (int)a.cache.fixed);
  const int tiles = (hi - lo + kTile - 1) / kTile;
  const T* kb = (const T*)a.cache.k.data + hk * a.cache.k.sh;
  const T* vb = (const T*)a.cache.v.data + hk * a.cache.v.sh;
  auto fetch = [&](int t) {
    if (t < tiles) {
      const uint32_t dst = sbase + (t % kStages) * 2 * TILE;
      constexpr int CH = D / 8;  // 16-byte pieces of a row
#pragma unroll
      for (int i = threadIdx.x; i < kTile * CH; i += kThreads) {
        const int key = i / CH, p = i - key * CH;
        const int at = lo + t * kTile + key;
        const int n = at < hi ? 16 : 0;  // zeros behind the end
        const int64_t g = min(at, hi - 1);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst + key * ROW + p * 16),
                     "l"(kb + g * a.cache.k.ss + p * 8), "r"(n)
                     : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst + TILE + key * ROW + p * 16),
                     "l"(vb + g * a.cache.v.ss + p * 8), "r"(n)
                     : "memory");
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
#pragma unroll
  for (int t = 0; t < kStages - 1; ++t) fetch(t);
  uint32_t q[NQ][STEPS][2];
  float o[NQ][STEPS][4], m[NQ][2], l[NQ][2];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = row0 + 8 * n + r;
    const int bb = row < a.rows ? row / a.group : 0, h = hk * a.group + (row < a.rows ? row - bb * a.group : 0);
    const T* qp = (const T*)a.q + bb * a.sqb + h * a.sqh + 2 * c;
#pragma unroll
    for (int t = 0; t < STEPS; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float e0 = row < a.rows ? to_f<T>(qp[16 * t + 8 * x]) : 0.f;
        const float e1 = row < a.rows ? to_f<T>(qp[16 * t + 8 * x + 1]) : 0.f;
        q[n][t][x] = Pair<T>::pack(e0, e1);
      }
#pragma unroll
    for (int t = 0; t < STEPS; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][t][e] = 0.f;
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
  }
  const uint32_t k_lane = ((lane & 7) + ((lane >> 3) & 1) * 8) * ROW + (lane >> 4) * 16;
  const uint32_t v_lane = ((lane & 7) + (lane >> 4) * 8) * ROW + ((lane >> 3) & 1) * 16;
#pragma unroll 1
  for (int t = 0; t < tiles; ++t) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 2) : "memory");
    __syncthreads();  // the tile is here for every warp, and the one before it is done with
    fetch(t + kStages - 1);
    const uint32_t ks = sbase + (t % kStages) * 2 * TILE, vs = ks + TILE;
    const int left = hi - lo - t * kTile;
#pragma unroll
    for (int g = 0; g < kTile / 16; ++g) {
      if (g * 16 >= left) break;
      float sc[NQ][4];
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        uint32_t f[4];
        ldmatrix4(f, ks + g * 16 * ROW + s * 32 + k_lane);
#pragma unroll
        for (int n = 0; n < NQ; ++n) Pair<T>::mma(sc[n], f[0], f[1], f[2], f[3], q[n][s][0], q[n][s][1]);
      }
      float grow = -INFINITY;
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[n][e] *= a.scale_log2;
          if (left < kTile && g * 16 + (e >> 1) * 8 + r >= left) sc[n][e] = -INFINITY;
          grow = fmaxf(grow, sc[n][e] - m[n][e & 1]);
        }
      if (__any_sync(0xffffffffu, grow > 8.f)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(m[n][e], fmaxf(sc[n][e], sc[n][2 + e]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            const float corr = mx == m[n][e] ? 1.f : ex2(m[n][e] - mx);
            m[n][e] = mx;
            l[n][e] *= corr;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
              o[n][s][e] *= corr;
              o[n][s][2 + e] *= corr;
            }
          }
      }
      uint32_t p[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            w[e] = ex2(sc[n][2 * h + e] - (m[n][e] == -INFINITY ? 0.f : m[n][e] - kAim<T>));
            l[n][e] += w[e];
          }
          p[n][h] = transpose8x8(Pair<T>::pack(w[0], w[1]));
        }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        uint32_t f[4];
        ldmatrix4_trans(f, vs + g * 16 * ROW + s * 32 + v_lane);
#pragma unroll
        for (int n = 0; n < NQ; ++n) Pair<T>::mma(o[n][s], f[0], f[1], f[2], f[3], p[n][0], p[n][1]);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
  wait_for_previous();
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[n][e];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      const int row = row0 + 8 * n + 2 * c + e;
      if (row >= a.rows) continue;
      const int bb = row / a.group, h = hk * a.group + row - bb * a.group;
      float* dst = a.part + (((int64_t)bb * a.Hq + h) * a.splits + a.split0 + split) * (D + 2);
      if (r == 0) {
        dst[D] = m[n][e] - kAim<T>;
        dst[D + 1] = sum;
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        dst[16 * s + r] = o[n][s][e];
        dst[16 * s + 8 + r] = o[n][s][2 + e];
      }
    }
}

// rows of a block of decode_prefix_kernel: 32 a warp where the accumulators fit the registers
int prefix_block_rows(int64_t rows, int64_t d) { return rows > 64 && d == 64 ? 128 : 64; }

template <typename T, int D, int NQ>
void launch_prefix_rows(const MmaArgs& a, int Hkv) {
  constexpr size_t smem = (size_t)kStages * 2 * kTile * (D * 2 + 16);
  C10_CUDA_CHECK(cudaFuncSetAttribute(decode_prefix_kernel<T, D, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int tiles = (a.rows + kWarps * 8 * NQ - 1) / (kWarps * 8 * NQ);
  launch(decode_prefix_kernel<T, D, NQ>, dim3((unsigned)(a.nsplit * tiles), (unsigned)Hkv), kThreads, smem, a.early, a);
}
template <typename T>
void launch_prefix(const MmaArgs& a, int Hkv, int d) {
  if (d == 64 && prefix_block_rows(a.rows, d) == 128)
    launch_prefix_rows<T, 64, 4>(a, Hkv);
  else if (d == 64)
    launch_prefix_rows<T, 64, 2>(a, Hkv);
  else if (d == 96)
    launch_prefix_rows<T, 96, 2>(a, Hkv);
  else
    launch_prefix_rows<T, 128, 2>(a, Hkv);
}

// 8 or 16 query rows a warp
template <typename T, typename C, int D>
void launch_rows(MmaArgs& a, int Hkv, int B) {
  a.tiles = (a.rows + 15) / 16;
  if (a.rows <= 8)
    launch_mma<T, C, D, 1>(a, Hkv, B);
  else
    launch_mma<T, C, D, 2>(a, Hkv, B);
}

template <typename T, typename C>
void launch_dim(MmaArgs& a, int Hkv, int B, int d) {
  if (d == 64)
    launch_rows<T, C, 64>(a, Hkv, B);
  else if (d == 96)
    launch_rows<T, C, 96>(a, Hkv, B);
  else
    launch_rows<T, C, 128>(a, Hkv, B);
}

bool mma_dim(int64_t d) { return d == 64 || d == 96 || d == 128; }

// 16-byte rows, which the tensor-core path loads
bool rows16(const CacheView& v, int64_t size) {
  return (uintptr_t)v.data % 16 == 0 && v.sb * size % 16 == 0 && v.sh * size % 16 == 0 && v.ss * size % 16 == 0;
}

template <typename T>
void launch_kind(MmaArgs& a, int kind, int Hkv, int B, int d) {
  if (kind == KV_I8)
    launch_dim<T, int8_t>(a, Hkv, B, d);
  else if (kind == KV_E4M3)
    launch_dim<T, e4m3>(a, Hkv, B, d);
  else
    launch_dim<T, T>(a, Hkv, B, d);
}

template <typename C, int LANES>
void launch_simt(const DecodeArgs& a) {
  const int G = a.group == 1 ? 1 : 4;
  const dim3 grid((unsigned)(a.nsplit * ((a.group + G - 1) / G)), (unsigned)a.Hkv, (unsigned)a.B);
  if (G == 1)
    launch(decode_simt_kernel<C, LANES, 1>, grid, kThreads, 0, a.early, a);
  else
    launch(decode_simt_kernel<C, LANES, 4>, grid, kThreads, 0, a.early, a);
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

// Pieces for `keys` keys a row: one round of the GPU at three blocks an SM, pieces
// of 128 to 1024 keys.  (The upper bound is for batches of unequal lengths: the
// longest sequence's blocks must not be the last ones running.)
// Up to 512 keys one piece saves the join.  In one piece / in several, 12 heads of
// 64 in bf16, under a graph: one user, 256 keys 4.5 / 6.0 us, 384 keys 6.1 / 6.1, 512
// keys 7.4 / 6.0 (less the second launch's share of an eager call); 8 users, 512
// keys 8.1 / 8.5, 640 keys 9.1 / 9.6, 768 keys 10.2 / 9.8, 1024 keys 12.6 / 10.5.
int pieces(int64_t keys, int64_t blocks) {
  if (keys <= 512) return 1;
  const int64_t want = 3 * num_sms() / blocks;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::max<int64_t>(want, (keys + 1023) / 1024), (keys + 127) / 128));
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
  const int kind = cache_kind(ck.scalar_type(), what);
  const bool half_q = a.q_type != KV_F32;
  const bool eight = kind == KV_I8 || kind == KV_E4M3;
  const bool mma_cache = half_q && mma_dim(d) && (eight || kind == a.q_type) && rows16(a.src.k, ck.element_size()) &&
                         rows16(a.src.v, ck.element_size());
  // A short prefix is seen by the cache's own kernel (16-bit kinds): one launch less.  A longer one is read once for
  // up to 128 query rows by the tensor-core path, once per sequence by the other.  Inline / in a launch of its own, ring
  // of 512 and 12 heads of 64 in bf16, under a graph: 4 tokens, one user 7.9 / 10.0 us, 64 users 22.6 / 25.1; 128 tokens
  // 8.8 / 10.0 and 24.9 / 24.9; 256 tokens 10.1 / 10.1 and 27.3 / 26.1; 512 tokens 12.6 / 11.1 and 32.2 / 26.2.
  const bool inline_prefix = has_prefix && mma_cache && !eight && P <= 128;
  const bool mma_prefix = half_q && mma_dim(d) && has_prefix && !inline_prefix;
  const int cs = pieces(std::min<int64_t>(S, window), B * Hkv);
  const int64_t prefix_rows = B * a.group;
  const bool many_rows = mma_prefix && prefix_rows > 16;
  int ps = 0;
  if (has_prefix && !inline_prefix) {
    const int64_t block_rows = many_rows ? prefix_block_rows(prefix_rows, d) : 16;
    const int64_t blocks = mma_prefix ? Hkv * ((prefix_rows + block_rows - 1) / block_rows) : B * Hkv;
    // many rows: a block a third of an SM, one round of the GPU, pieces of whole tiles
    ps = many_rows ? (int)std::max<int64_t>(1, std::min<int64_t>(3 * num_sms() / blocks, (P + 255) / 256)) : pieces(P, blocks);
  }
  a.splits = cs + ps;
  at::Tensor part;
  if (a.splits > 1 || !mma_cache) {
    part = at::empty({B * Hq, a.splits, d + 2}, q.options().dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  MmaArgs m{};
  m.q = a.q;
  m.sqb = a.sqb;
  m.sqh = a.sqh;
  m.part = a.part;
  m.out = out.data_ptr();
  m.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  m.splits = a.splits;
  m.Hq = a.Hq;
  m.group = a.group;
  m.scale_log2 = a.scale_log2;
  auto run_mma = [&](int k) {
    if (a.q_type == KV_BF16)
      launch_kind<__nv_bfloat16>(m, k, a.Hkv, a.B, a.d);
    else
      launch_kind<__half>(m, k, a.Hkv, a.B, a.d);
    check_launch(what);
  };
  if (inline_prefix) {
    m.ahead.k = prefix_view(*pk, hold_pk);
    m.ahead.v = prefix_view(*pv, hold_pv);
    m.ahead.fixed = P;
    m.ahead.S = 1 << 30;
  } else if (has_prefix) {
    DecodeArgs p = a;
    p.src.k = prefix_view(*pk, hold_pk);
    p.src.v = prefix_view(*pv, hold_pv);
    p.src.lengths = nullptr;
    p.src.fixed = P;
    p.src.S = 1 << 30;
    p.nsplit = ps;
    p.split0 = 0;
    if (mma_prefix) {
      m.cache = p.src;
      m.rows = (int)prefix_rows;
      m.shared = true;
      m.split0 = 0;
      m.nsplit = ps;
      m.piece = (int)((P + ps - 1) / ps);
      if (many_rows) {
        m.piece = (m.piece + kTile - 1) / kTile * kTile;
        if (a.q_type == KV_BF16)
          launch_prefix<__nv_bfloat16>(m, a.Hkv, a.d);
        else
          launch_prefix<__half>(m, a.Hkv, a.d);
        check_launch(what);
      } else {
        run_mma(a.q_type);
      }
    } else {
      launch_source(p, a.q_type);
      check_launch(what);
    }
  }
  a.nsplit = cs;
  a.split0 = ps;
  a.early = m.early = ps > 0;
  if (mma_cache) {
    m.cache = a.src;
    m.rows = a.group;
    m.shared = false;
    m.split0 = ps;
    m.nsplit = cs;
    m.piece = (int)((std::min<int64_t>(S, window) + cs - 1) / cs);
    run_mma(kind);
    if (a.splits == 1) return {out, lse};
  } else {
    launch_source(a, kind);
    check_launch(what);
  }
  const int64_t rows = B * Hq;
  TORCH_CHECK(rows < (1ll << 31), what, ": too many query rows in one call");
  TB_DISPATCH_FLOAT(q.scalar_type(), what, [&] {
    launch(decode_join_kernel<scalar_t>, dim3((unsigned)rows), 32 * kJoinWarps, 0, true, a.part, a.splits, (int)d,
           (scalar_t*)out.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr);
  });
  check_launch(what);
  return {out, lse};
}

}  // namespace tb
