// Log probabilities of given tokens, entropy, log-sum-exp and the k most probable tokens of rows of logits, and the gradient of the first
// two (include/crl.h: crl_token_logprobs, crl_token_logprobs_bwd).
//   m = max x, S = sum 2^t, T = sum t 2^t with t = (x - m) log2(e):  lse = m + ln S,  H = ln 2 (log2 S - T / S),  log p_j = (x_j - m) - ln S
// all in fp32; the deviations t are taken before anything is summed, so neither H nor log p is a difference of large numbers.  The gradient takes log p_j
// as x_j - lse: exact but for the rounding of lse to fp32, so log p, and relatively p, are off by 2^-24 |lse| there.
#include "common.h"

namespace {

constexpr float L2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;
constexpr int TOP_MAX = 32;
constexpr int CAND = 512;               // candidates that the selecting wave looks at; more: the slow path

template <typename T> struct Vec;       // 16 bytes of logits
template <> struct Vec<u16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(const u32x4& v, int j) {
    const uint32_t w = v[j >> 1];
    return __uint_as_float((j & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ float pick(const u32x4& v, int j) {
    const uint32_t w = j < 2 ? v[0] : j < 4 ? v[1] : j < 6 ? v[2] : v[3];
    return __uint_as_float((j & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  // columns from `n` on become -inf
  static __device__ __forceinline__ void cut(u32x4& w, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 2 * i >= n ? 0xff80ff80u : 2 * i + 1 >= n ? (w[i] & 0xffffu) | 0xff800000u : w[i];
  }
  // the n columns from p on and -inf behind them, read one by one
  static __device__ __forceinline__ u32x4 tail(const u16* p, int n) {
    u32x4 v{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) v[j >> 1] = (j & 1) ? (v[j >> 1] & 0xffffu) | bits_of(p[j]) << 16 : (v[j >> 1] & 0xffff0000u) | bits_of(p[j]);
    return v;
  }
  static __device__ __forceinline__ uint32_t bits_of(u16 x) { return x; }
  static __device__ __forceinline__ void put(u16* p, const u32x4& v, int j) { *p = (u16)(v[j >> 1] >> 16 * (j & 1)); }
};
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(const u32x4& v, int j) { return __uint_as_float(v[j]); }
  static __device__ __forceinline__ float pick(const u32x4& v, int j) { return __uint_as_float(j < 1 ? v[0] : j < 2 ? v[1] : j < 3 ? v[2] : v[3]); }
  static __device__ __forceinline__ void cut(u32x4& w, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = i >= n ? 0xff800000u : w[i];
  }
  static __device__ __forceinline__ u32x4 tail(const float* p, int n) {
    u32x4 v{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) v[j] = __float_as_uint(p[j]);
    return v;
  }
  static __device__ __forceinline__ void put(float* p, const u32x4& v, int j) { *p = __uint_as_float(v[j]); }
};
// NT: past the caches
template <bool NT>
__device__ __forceinline__ u32x4 load16(const void* p) {
  return NT ? __builtin_nontemporal_load((const u32x4*)p) : *(const u32x4*)p;
}
__device__ __forceinline__ float load1(const u16* p) { return bf2f(*p); }
__device__ __forceinline__ float load1(const float* p) { return *p; }

struct LpArgs {
  const void* logits; int64_t ldl;
  const int64_t* target;
  float *logprob, *entropy, *lse, *top_lp;
  int64_t* top_ids;
  int64_t top_ld, ids_ld;
  int64_t M;
  int V, k;
};

// (value, token) in one whole number: larger value first, of equal values the lower token; NaN above everything, -0 with +0
__device__ __forceinline__ uint64_t cand_key(float x, int idx) {
  uint32_t u = __float_as_uint(x + 0.f);
  u = !(x == x) ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)(0x7fffffff - idx);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_token(uint64_t key) { return 0x7fffffff - (int)(uint32_t)key; }

// reductions over the 64 lanes on the DPP path (shifts within rows of 16, then broadcasts of rows): about 50 cycles where six LDS permutes
// take 600; the result sits in lane 63 and is read from there into a scalar
template <int CTRL, int ROWS, typename F>
__device__ __forceinline__ float dpp_step(float v, float none, F f) {
  return f(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false)));
}
template <typename F>
__device__ __forceinline__ float dpp_reduce(float v, float none, F f) {
  v = dpp_step<0x111, 0xf>(v, none, f);
  v = dpp_step<0x112, 0xf>(v, none, f);
  v = dpp_step<0x114, 0xf>(v, none, f);
  v = dpp_step<0x118, 0xf>(v, none, f);
  v = dpp_step<0x142, 0xa>(v, none, f);
  v = dpp_step<0x143, 0xc>(v, none, f);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float max_all(float v) { return dpp_reduce(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float sum_all(float v) { return dpp_reduce(v, 0.f, [](float a, float b) { return a + b; }); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_step64(uint64_t v) {
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint64_t x = ((uint64_t)hi << 32) | lo;
  return x > v ? x : v;
}
__device__ __forceinline__ uint64_t max_all64(uint64_t v) {
  v = dpp_step64<0x111, 0xf>(v);
  v = dpp_step64<0x112, 0xf>(v);
  v = dpp_step64<0x114, 0xf>(v);
  v = dpp_step64<0x118, 0xf>(v);
  v = dpp_step64<0x142, 0xa>(v);
  v = dpp_step64<0x143, 0xc>(v);
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}

// sums taken against the reference `from` -> the same against `to` >= from.  A factor that underflows leaves zeros: `from` may be the lowest
// finite value (masked columns seen first), and then the distance is infinite
__device__ __forceinline__ void shift(float& S, float& T, float from, float to) {
  const float d = (from - to) * L2E, al = __builtin_amdgcn_exp2f(d);
  T = al == 0.f ? 0.f : al * __builtin_fmaf(d, S, T);
  S *= al;                                                 // (NaN stays NaN)
}

// One workgroup of NT threads per row.  A thread walks its 16-byte pieces U at a time, the next U on their way, with a maximum and sums of its
// own: no barrier until the row has been read.  The logits are read once, and bound it: 8184 x 50304 bf16, 823 MB in 151 us, 5.45 TB/s
// (a copy of that size reaches 5.05; the first hundred calls up to 190), without top tokens 147, with masked columns 178 to 195 (the exponentials of a
// batch that holds a mask are computed twice); 8 rows of 50267, 9.9 us, are latency: launch, 6 pieces a thread, three exchanges, the candidates' second look.
// The k best: the k-th largest of the maxima of 64 groups of lanes is a bound that the k-th best cannot be under.  The lanes whose maximum
// reaches it (about k of them) read the pieces around it once more (all of theirs where the second largest reaches it too) and put what reaches it
// into a list in LDS that the first wave picks from.  Rows of many equal values overflow the list and take k rounds over the row instead.
template <typename T, int NT, int U, bool TOP>
__global__ __launch_bounds__(NT) void logprobs_kernel(const LpArgs a) {
  constexpr int N = Vec<T>::N, NW = NT / 64;
  __shared__ float red[3][NW];
  __shared__ uint64_t list[TOP ? CAND : 1], best[TOP ? TOP_MAX : 1], best_of[NW];
  __shared__ float gmax[64];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.logits + row * a.ldl;
  const int V = a.V;
  const int pieces = (V + N - 1) / N, whole = V / N;
  const int64_t tgt = a.logprob ? a.target[row] : -100;
  const bool inside = tgt >= 0 && tgt < V;
  const float xt = inside ? load1(x + tgt) : 0.f;
  float m = -INFINITY, S = 0.f, TT = 0.f;
  float second = -INFINITY;                                // the largest logit outside the U pieces from at_max on, which hold m
  int at_max = tid;

  // Where V is no multiple of N, piece `whole` reaches past it: into the row's padding, or, in the last row, perhaps out of the matrix.  There its
  // thread reads it by columns, beforehand.
  const bool end = row == a.M - 1;
  const int full = end ? whole : pieces;                   // pieces that may be read as such
  u32x4 part = Vec<T>::tail(x, 0);
  if (end && tid == whole % NT) part = Vec<T>::tail(x + (int64_t)whole * N, V - whole * N);
  const auto piece = [&](int p) {
    u32x4 v = part;
    if (p < full) {
      v = *reinterpret_cast<const u32x4*>(x + (int64_t)p * N);
      if (p >= whole) Vec<T>::cut(v, V - p * N);
    }
    return v;
  };
  u32x4 nx[U];
#pragma unroll
  for (int u = 0; u < U; ++u) nx[u] = full ? *reinterpret_cast<const u32x4*>(x + (int64_t)min(tid + u * NT, full - 1) * N) : part;
  for (int p0 = tid; p0 < pieces; p0 += NT * U) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = nx[u];
      if (full) nx[u] = *reinterpret_cast<const u32x4*>(x + (int64_t)min(p0 + (U + u) * NT, full - 1) * N);
    }
    if (p0 + (U - 1) * NT >= whole) {                      // columns past V count as -inf
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int p = p0 + u * NT;
        if (p == whole && end) v[u] = part;
        else if (p >= whole) Vec<T>::cut(v[u], V - p * N);
      }
    }
    float f[U * N];
#pragma unroll
    for (int i = 0; i < U * N; ++i) f[i] = Vec<T>::get(v[i / N], i % N);
    float mx = f[0];
#pragma unroll
    for (int i = 1; i < U * N; ++i) mx = fmaxf(mx, f[i]);
    if (mx > m) {                                          // (a row of -inf only keeps m = -inf and S = 0: NaN at the end)
      shift(S, TT, m, mx);
      second = m;
      m = mx;
      at_max = p0;
    } else {
      second = fmaxf(second, mx);
    }
    const float ref = m == -INFINITY ? 0.f : m, T0 = TT;
#pragma unroll
    for (int i = 0; i < U * N; ++i) {
      const float t = (f[i] - ref) * L2E, e = __builtin_amdgcn_exp2f(t);
      S += e;
      TT = __builtin_fmaf(t, e, TT);                       // NaN where t = -inf and e = 0: put right below
    }
    if (__any(!(TT == TT))) {                              // -inf among the logits (or NaN, which S keeps); rare, and too long to compute beside
      TT = T0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        asm volatile("" : "+v"(v[u]));
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float t = (Vec<T>::get(v[u], j) - ref) * L2E;
          TT = __builtin_fmaf(fmaxf(t, -1e30f), __builtin_amdgcn_exp2f(t), TT);
        }
      }
    }
  }
  if (TOP) {
    const int k = a.k;
    float g = m;
#pragma unroll
    for (int o = 1; o < NW; o <<= 1) g = fmaxf(g, __shfl_xor(g, o, 64));
    if ((lane & (NW - 1)) == 0) gmax[tid / NW] = g;
    if (tid == 0) count = 0;
    __syncthreads();
    float thr = INFINITY;
    {
      float gv = gmax[lane];
      for (int i = 0; i < k; ++i) {
        thr = max_all(gv);
        const unsigned long long who = __ballot(gv == thr);
        if (who && lane == __ffsll(who) - 1) gv = -INFINITY;
      }
    }
    if (m >= thr || !(S == S)) {                           // NaN counts as largest: every list is filled with tokens of the row
      const bool one = second < thr && S == S;             // nearly always: then the pieces around the maximum are all there is to read
      for (int p0 = one ? at_max : tid; p0 < pieces; p0 = one ? pieces : p0 + NT * U) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = piece(p0 + u * NT);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c0 = (p0 + u * NT) * N;
          uint32_t hits = 0;
#pragma unroll
          for (int j = 0; j < N; ++j) hits |= (c0 + j < V && !(Vec<T>::get(v[u], j) < thr)) ? 1u << j : 0u;
          while (hits) {
            const int j = __ffs(hits) - 1;
            hits &= hits - 1;
            const int at = atomicAdd(&count, 1);
            if (at < CAND) list[at] = cand_key(Vec<T>::pick(v[u], j), c0 + j);
          }
        }
      }
    }
    __syncthreads();
    const int total = count;
    if (total <= CAND) {
      if (wave == 0) {
        const uint64_t c = lane < total ? list[lane] : 0;
        uint64_t prev = ~0ull;
        for (int i = 0; i < k; ++i) {
          uint64_t b = c < prev ? c : 0;
          for (int q = 64 + lane; q < total; q += 64) {
            const uint64_t y = list[q];
            if (y < prev && y > b) b = y;
          }
          prev = max_all64(b);
          if (lane == 0) best[i] = prev;
        }
      }
    } else {
      uint64_t prev = ~0ull;
      for (int i = 0; i < k; ++i) {
        uint64_t b = 0;
        for (int p = tid; p < pieces; p += NT) {
          const u32x4 u = piece(p);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const uint64_t c = cand_key(Vec<T>::get(u, j), p * N + j);
            if (p * N + j < V && c < prev && c > b) b = c;
          }
        }
        b = max_all64(b);
        if (lane == 0) best_of[wave] = b;
        __syncthreads();
        b = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) b = best_of[w] > b ? best_of[w] : b;
        __syncthreads();
        if (tid == 0) best[i] = b;
        prev = b;
      }
    }
  }
  // lanes -> wave -> workgroup
  {
    const float mw = max_all(m);
    if (m != -INFINITY) shift(S, TT, m, mw);               // (m = -inf: nothing to scale, or NaN that stays)
    S = sum_all(S);
    TT = sum_all(TT);
    if (lane == 0) { red[0][wave] = mw; red[1][wave] = S; red[2][wave] = TT; }
  }
  __syncthreads();
  if (wave != 0) return;
  float mg = -INFINITY, Sg = 0.f, Tg = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) mg = fmaxf(mg, red[0][w]);
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    float Sw = red[1][w], Tw = red[2][w];
    if (red[0][w] != -INFINITY) shift(Sw, Tw, red[0][w], mg);
    Sg += Sw;
    Tg += Tw;
  }
  const bool none = mg == -INFINITY;                       // no finite logit: there is no distribution
  const float lnS = none ? __builtin_nanf("") : logf(Sg);
  if (lane == 0) {
    if (a.lse) a.lse[row] = none ? (Sg == 0.f ? -INFINITY : __builtin_nanf("")) : mg + lnS;
    if (a.entropy) a.entropy[row] = none ? __builtin_nanf("") : lnS - LN2 * (Tg / Sg);
    if (a.logprob) a.logprob[row] = tgt == -100 ? 0.f : !inside ? __builtin_nanf("") : (xt - mg) - lnS;
  }
  if (TOP && lane < a.k) {
    const uint64_t c = best[lane];
    a.top_ids[row * a.ids_ld + lane] = key_token(c);
    a.top_lp[row * a.top_ld + lane] = (key_value(c) - mg) - lnS;
  }
}

struct LpBwdArgs {
  const void* logits; void* dlogits; int64_t ldl, ldd;
  const int64_t* target;
  const float *lse, *entropy, *d_logprob, *d_entropy;
  int64_t M;
  int V, cols;
};

__device__ __forceinline__ u32x4 pack16(const float (&o)[8]) { return u32x4{pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]), pack_bf2(o[4], o[5]), pack_bf2(o[6], o[7])}; }
__device__ __forceinline__ u32x4 pack16(const float (&o)[4]) { return u32x4{__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])}; }

// d x_j = g (1[j = t] - p_j) - gH p_j (log p_j + H); p_j = 0 takes its limit 0. one workgroup per row and 256 * BWD_U pieces; columns from V on zeroed.
// lse and H are the forward's, so a logit needs no other: read once, written once.  8184 x 50304 bf16: 1.65 GB in 315 us, 5.24 TB/s;
// right behind the forward call, which leaves a part of the logits in the last cache, 280
constexpr int BWD_U = 4;                // 16-byte loads in flight per thread
template <typename T, bool FAR>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(const LpBwdArgs a) {
  constexpr int N = Vec<T>::N;
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.logits + row * a.ldl;
  T* d = (T*)a.dlogits + row * a.ldd;
  const int64_t t = a.target ? a.target[row] : -100;
  const bool invalid = t != -100 && (t < 0 || t >= a.V);
  float g = a.d_logprob && t != -100 ? a.d_logprob[row] : 0.f;
  if (invalid) g = __builtin_nanf("");
  const float gh = a.d_entropy ? a.d_entropy[row] : 0.f;
  const float H = a.d_entropy ? a.entropy[row] : 0.f;
  const float lse = a.lse[row];
  const float c0 = __builtin_fmaf(gh, H, g);               // d x_j = -p_j (c0 + gH log p_j) + g 1[j = t]
  const int V = g == 0.f && gh == 0.f ? 0 : a.V;           // a row that takes no gradient is not read: zeros, also where it holds no distribution
  const int pieces = (a.cols + N - 1) / N, whole = V / N;
  const int full = row == a.M - 1 ? whole : (V + N - 1) / N;                // pieces that may be read as such
  const int p0 = blockIdx.y * (256 * BWD_U) + threadIdx.x;
  u32x4 v[BWD_U] = {};
  if (full) {
#pragma unroll
    for (int u = 0; u < BWD_U; ++u) v[u] = load16<FAR>(x + (int64_t)min(p0 + u * 256, full - 1) * N);
  }
  if (row == a.M - 1) {                                    // the last piece of the last row may reach out of the matrix: by columns
#pragma unroll
    for (int u = 0; u < BWD_U; ++u)
      if (p0 + u * 256 == whole) v[u] = Vec<T>::tail(x + (int64_t)whole * N, V - whole * N);
  }
#pragma unroll
  for (int u = 0; u < BWD_U; ++u) {
    const int p = p0 + u * 256;
    if (p >= pieces) break;
    float o[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float lp = Vec<T>::get(v[u], j) - lse;
      const float e = __builtin_amdgcn_exp2f(lp * L2E);
      float r = -e * __builtin_fmaf(gh, lp, c0);
      if (e == 0.f) r = 0.f;
      if (p * N + j == (int)t) r += g;
      o[j] = p * N + j < V ? r : 0.f;
    }
    const u32x4 r = pack16(o);
    if (p * N + N > a.cols) {                              // a part of a piece: column by column
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (p * N + j < a.cols) Vec<T>::put(d + (int64_t)p * N + j, r, j);
    } else if (FAR) {
      __builtin_nontemporal_store(r, reinterpret_cast<u32x4*>(d + (int64_t)p * N));
    } else {
      *reinterpret_cast<u32x4*>(d + (int64_t)p * N) = r;
    }
  }
}

template <typename T, int NT, int U>
void launch_lp(const LpArgs& a, hipStream_t s) {
  const unsigned g = (unsigned)a.M;
  if (a.k) logprobs_kernel<T, NT, U, true><<<g, NT, 0, s>>>(a);
  else logprobs_kernel<T, NT, U, false><<<g, NT, 0, s>>>(a);
}

}  // namespace

extern "C" int crl_token_logprobs(const void* logits, int is_f32, int64_t ldl, const int64_t* target, int64_t M, int V, float* logprob,
                                  float* entropy, float* lse, int k, float* top_logprob, int64_t top_ld, int64_t* top_ids, int64_t ids_ld,
                                  void* stream) {
  const char* who = "crl_token_logprobs";
  CRL_CHECK(logits, "%s: null pointer", who);
  CRL_CHECK(M > 0 && M < (1ll << 31) && V > 0 && V < (1 << 30), "%s: bad shape M=%lld V=%d", who, (long long)M, V);
  const int vec = is_f32 ? 4 : 8;
  CRL_CHECK(((uintptr_t)logits % 16) == 0 && (M == 1 || (ldl % vec == 0 && ldl >= V)),
            "%s: rows must start 16-byte aligned and hold V = %d columns (ldl = %lld)", who, V, (long long)ldl);
  CRL_CHECK((logprob != nullptr) == (target != nullptr), "%s: logprob and target go together", who);
  CRL_CHECK(logprob || entropy || lse || k, "%s: nothing to compute", who);
  CRL_CHECK(k >= 0 && k <= TOP_MAX && k <= V, "%s: top %d of %d tokens (at most %d)", who, k, V, TOP_MAX);
  CRL_CHECK(k == 0 || (top_logprob && top_ids && top_ld >= k && ids_ld >= k), "%s: top_logprob and top_ids need %d columns", who, k);
  LpArgs a{logits, ldl, target, logprob, entropy, lse, top_logprob, top_ids, top_ld, ids_ld, M, V, k};
  hipStream_t s = as_stream(stream);
  // Threads a row: a wave for short rows; 1024 where there are fewer rows than places for workgroups and only latency counts; 256 elsewhere, eight rows
  // a CU in different phases.  256 against 1024 threads, rows of 50267 bf16, the best token, in us: 8 rows 10.5 / 8.2, 128 11.3 / 9.0, 256 13.3 / 10.1,
  // 384 15.1 / 14.7, 512 18.0 / 15.3, 768 21.5 / 22.8, 1024 25.2 / 28.2, 2048 45.3 / 50.7, 8184 151 / 175; 8 rows of 4096 4.8 / 4.7, 8192 5.2 / 5.2,
  // 16384 6.1 / 5.7.
  const int pieces = (V + vec - 1) / vec;
  if (pieces <= 128) { if (is_f32) launch_lp<float, 64, 2>(a, s); else launch_lp<u16, 64, 2>(a, s); }
  else if (M >= 512 || pieces <= 1024) { if (is_f32) launch_lp<float, 256, 2>(a, s); else launch_lp<u16, 256, 2>(a, s); }
  else { if (is_f32) launch_lp<float, 1024, 1>(a, s); else launch_lp<u16, 1024, 1>(a, s); }
  CRL_LAUNCH_CHECK(who);
  return 0;
}

extern "C" int crl_token_logprobs_bwd(const void* logits, int is_f32, int64_t ldl, const int64_t* target, int64_t M, int V, const float* lse,
                                      const float* entropy, const float* d_logprob, const float* d_entropy, void* dlogits, int64_t ldd, int cols,
                                      void* stream) {
  const char* who = "crl_token_logprobs_bwd";
  CRL_CHECK(logits && lse && dlogits, "%s: null pointer", who);
  CRL_CHECK(d_logprob || d_entropy, "%s: neither d_logprob nor d_entropy", who);
  CRL_CHECK(!d_logprob || target, "%s: d_logprob needs target", who);
  CRL_CHECK(!d_entropy || entropy, "%s: d_entropy needs entropy", who);
  CRL_CHECK(M > 0 && M < (1ll << 31) && V > 0 && V < (1 << 30), "%s: bad shape M=%lld V=%d", who, (long long)M, V);
  const int vec = is_f32 ? 4 : 8;
  CRL_CHECK(cols >= V && cols < (1 << 30) && ((uintptr_t)logits % 16) == 0 && ((uintptr_t)dlogits % 16) == 0 &&
                (M == 1 || (ldl % vec == 0 && ldd % vec == 0 && ldl >= V && ldd >= cols)),
            "%s: rows must start 16-byte aligned and hold V = %d (cols = %d) columns (ldl = %lld, ldd = %lld)", who, V, cols, (long long)ldl,
            (long long)ldd);
  CRL_CHECK(dlogits != logits || ldd == ldl, "%s: in place with another row stride", who);
  LpBwdArgs a{logits, dlogits, ldl, ldd, d_logprob ? target : nullptr, lse, entropy, d_logprob, d_entropy, M, V, cols};
  const dim3 grid((unsigned)M, (unsigned)(((cols + vec - 1) / vec + 256 * BWD_U - 1) / (256 * BWD_U)));
  CRL_CHECK(grid.y < 65536, "%s: too many columns (%d)", who, cols);
  // Past the caches where the logits are larger than the last of them (256 MiB): nobody finds a line again, and keeping them costs evictions
  // (8184 x 50304 bf16: 315 us against 329, behind the forward call both together 425 against 488; 127 x 50304 fp32, both calls: 19.8 against 18.8 with
  // three sets of logits in turn, 21.0 against 22.4 with twelve, so no rule there).
  const bool far = (size_t)M * ldl * (is_f32 ? 4 : 2) > (256u << 20);
  hipStream_t s = as_stream(stream);
  if (is_f32) { if (far) logprobs_bwd_kernel<float, true><<<grid, 256, 0, s>>>(a); else logprobs_bwd_kernel<float, false><<<grid, 256, 0, s>>>(a); }
  else { if (far) logprobs_bwd_kernel<u16, true><<<grid, 256, 0, s>>>(a); else logprobs_bwd_kernel<u16, false><<<grid, 256, 0, s>>>(a); }
  CRL_LAUNCH_CHECK(who);
  return 0;
}
