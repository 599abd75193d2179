// A key-value cache in pages (include/crl.h: crl_paged_attn_decode, crl_paged_append, crl_cache_evict), head_dim 64, bf16.
// Position p of sequence b lives in slot p % page_size of page page_table[b][p / page_size] of one pool; sequences have lengths of their
// own in device memory, so that one captured graph serves every step.  A page id outside the pool or a length outside the table never
// becomes an address: the rows of such a sequence come out NaN (attention) or stay as they are (append, evict).
#include "common.h"

namespace {

constexpr float LOG2E_P = 1.4426950408889634f;
constexpr int PART = 66;                // floats of a partial result in memory: m, l, o[64]
constexpr int RED = 68;                 // floats between the partial results of a wave's heads in LDS
constexpr int HEADS = 16;               // query heads of a workgroup
constexpr int MAX_SPLIT = 256;
constexpr int W_DIRECT = 16384;         // positions x query heads a key-value head up to which one launch also adds the weights

// position -> offset of its row (elements) from the base of a head's rows
struct Pages {
  const int* table;                     // [B][table_ld]
  int64_t table_ld;
  int64_t page_s, row_s, head_s;        // strides of the pool in elements
  int n_pages, shift, cap;              // pages in the pool, log2(page size), positions a sequence's table row covers
};

// the row of position p, or false where the table holds no page of the pool (the offset is then page 0's, for a load that is not used)
__host__ __device__ __forceinline__ bool row_of(const Pages& pg, const int* table_row, int p, int64_t& off) {
  int id = table_row[p >> pg.shift];
  const bool ok = (unsigned)id < (unsigned)pg.n_pages;
  if (!ok) id = 0;
  off = id * pg.page_s + (p & ((1 << pg.shift) - 1)) * pg.row_s;
  return ok;
}

struct PagedArgs {
  const u16 *q, *k_new, *v_new;
  u16 *k, *v, *o;
  int64_t q_s, o_s, kn_s, vn_s;
  Pages pg;
  const int* lengths;
  float* weights; int64_t w_bs, w_hs;
  float* ws;                            // [B * H][nsplit][PART]
  float* scores;                        // [B * H][score_ld] base-2 logits, where the weights are asked for
  int64_t score_ld;
  int B, H, Hkv, group, nsub, nsplit, nw, kw_max;          // nw: waves of a workgroup of the attending launch
  int turn;                             // workgroups of split s begin `turn * s` (sequence, head) pairs further on
  float scale;
};

// Keys that a wave takes, whole batches, the same in the attending and in the joining launch.  Splits are of one size whatever the sequence's
// length (kw_max, the capacity over all waves of a sequence): long sequences have more of them, and workgroups do equal work in a ragged
// batch (32 sequences of 0 to 6189 keys, 16 query heads on 4: 29 us against 34 with every sequence cut into 8, before `turn`).  What fits one workgroup is
// spread over its waves.
__device__ __forceinline__ int keys_per_wave(int n, int nw, int kw_max) {
  return min(kw_max, max(64, ((n + nw - 1) / nw + 63) & ~63));
}
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// One workgroup = up to 16 query heads that share a key-value head x one split of a sequence's keys; every wave has its own
// range of them, in batches of 64.
// S^T = K Q^T and O^T += V^T P^T on the matrix cores (16x16x32): a lane holds ONE query (lane & 15) throughout, its scores of keys 16 t + 4 g + r
// (g = lane >> 4) and its output channels 16 c + 4 g + r, so maximum, sum and rescaling never leave it but for the maximum over the four g.
// K rows, then V rows go through the wave's own 8 KiB of LDS (16-byte chunks at chunk ^ (row & 7)), whole rows of memory an instruction, and come
// back as operands: K by rows, V transposed (ds_read_b64_tr_b16).  The key order of P V is that of the scores' registers: P needs no exchange.
// The probabilities enter P V as the sum of two bf16 numbers of their sign.  The first is 0.9961 p rounded, by half a step (2^-8) at most: under p.  The
// second is the rest, over 0 and up to 2^-7 of p, rounded by 2^-8 of itself: p is off by 2^-15 of itself at most, which the bf16 rounding of the
// output (2^-8) hides.  Neither is 0 or negative where p is not (down to 2^-109, where the rest is a normal number still), so an infinite value gives infinity.  All else is fp32.
// Bound by the key and value rows, read once from HBM and by nobody again: 8 sequences of 24935 keys, 16 heads: 818 MB in 144 us, 5.7 TB/s
// (random 8 KiB reads alone reach 5.85, a copy of 1 GB 5.05); 32 sequences of up to 6189 keys, 16 query heads on 4: 102 MB in 22 us.  The latter's
// vector units have 16 scores per key to exponentiate; where heads share keys, the matrix cores take the products from them (with dot products on the
// vector units that call took 46 us against 29).  Batches of 64 keys: the next batch's rows fly while this one is computed, 4 waves a SIMD.
// With weights the scores go to memory as well (and the registers' limit is 3 waves a SIMD): 6189 keys, 8 x 16 heads, 43 us of the call's 48.
template <int NW, bool W>
__global__ __launch_bounds__(64 * NW, W ? 3 : 4) void paged_attn_kernel(const PagedArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[NW][8192];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i = lane & 15;
  const int split = blockIdx.y;
  unsigned x = blockIdx.x;
  if (split) x = (x + split * a.turn) % gridDim.x;
  const int sub = x % a.nsub, bh = x / a.nsub;
  const int b = bh / a.Hkv, hk = bh % a.Hkv;
  const int h0 = hk * a.group + sub * HEADS;                 // first query head of this workgroup
  const int gn = min(HEADS, a.group - sub * HEADS);
  const int* table = a.pg.table + b * a.pg.table_ld;
  int page = 0;                                              // page of key base + lane; of the first wave's before the length is known
  if (split == 0 && wave == 0) page = table[min(lane, a.pg.cap - 1) >> a.pg.shift];
  const u16* qrow = a.q + b * a.q_s + (h0 + min(i, gn - 1)) * 64 + 8 * g;
  const bf16x8 q0 = *reinterpret_cast<const bf16x8*>(qrow), q1 = *reinterpret_cast<const bf16x8*>(qrow + 32);
  const bool has_new = a.k_new != nullptr;
  const int part = lane & 7, kr = lane >> 3;                 // loads: eight lanes a row, eight rows an instruction
  u32x4 kn, vn;                                              // this lane's 16 bytes of the appended row
  if (has_new) {
    kn = *reinterpret_cast<const u32x4*>(a.k_new + b * a.kn_s + hk * 64 + 8 * part);
    vn = *reinterpret_cast<const u32x4*>(a.v_new + b * a.vn_s + hk * 64 + 8 * part);
  }
  const int n_raw = a.lengths[b];
  bool bad = n_raw < 0 || n_raw > a.pg.cap;
  const int n = bad ? 0 : n_raw, nold = n - (has_new && n > 0 ? 1 : 0);
  const int kw = keys_per_wave(n, NW, a.kw_max);
  if (split * NW * kw >= n && split > 0 && !bad) return;     // (the joining launch does not look for these)
  const int k_lo = (split * NW + wave) * kw, k_hi = min(n, k_lo + kw);
  const float c = a.scale * LOG2E_P;
  u16* kb = a.k + hk * a.pg.head_s + 8 * part;
  u16* vb = a.v + hk * a.pg.head_s + 8 * part;
  if (has_new && split == 0 && wave == 0 && n > 0) {         // the appended row into its page (nothing of this call reads it there)
    int64_t off;
    if (!row_of(a.pg, table, n - 1, off)) bad = true;
    else if (sub == 0 && kr == 0) {
      *reinterpret_cast<u32x4*>(kb + off) = kn;
      *reinterpret_cast<u32x4*>(vb + off) = vn;
    }
  }

  char* tile = lds[wave];
  float m = -INFINITY, l = 0.f;
  f32x4 acc[4];
#pragma unroll
  for (int cg = 0; cg < 4; ++cg) acc[cg] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (k_lo > 0 && k_lo < k_hi) page = table[min(k_lo + lane, a.pg.cap - 1) >> a.pg.shift];

  for (int base = k_lo; base < k_hi; base += 64) {
    const int last = min(nold, k_hi) - 1 - base;             // last key of the pages, relative to the batch; < 0: the batch is the appended row
    u32x4 kv[8], vv[8];
    if (last >= 0) {
      if (lane <= last && (unsigned)page >= (unsigned)a.pg.n_pages) { bad = true; page = 0; }
      const int64_t my_off = page * a.pg.page_s + ((base + lane) & ((1 << a.pg.shift) - 1)) * a.pg.row_s;
      const int off_lo = (int)(uint32_t)my_off, off_hi = (int)(my_off >> 32);
      if (base + 64 < k_hi) page = table[min(base + 64 + lane, a.pg.cap - 1) >> a.pg.shift];
      int64_t off[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {                          // rows past the end of the pages: the last row again
        const int from = min(8 * j + kr, last);
        off[j] = ((int64_t)__shfl(off_hi, from, 64) << 32) | (uint32_t)__shfl(off_lo, from, 64);
        kv[j] = *reinterpret_cast<const u32x4*>(kb + off[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) vv[j] = *reinterpret_cast<const u32x4*>(vb + off[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) { kv[j] = kn; vv[j] = vn; }
    }
    if (base + 64 > min(nold, k_hi)) {                       // the last batch: the appended row in its place, zeros behind it
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = base + 8 * j + kr;
        if (has_new && key == nold) { kv[j] = kn; vv[j] = vn; }
        if (key >= k_hi) vv[j] = u32x4{0, 0, 0, 0};
      }
    }
    // (rows 8 j + kr have row & 7 = kr)
#pragma unroll
    for (int j = 0; j < 8; ++j) *reinterpret_cast<u32x4*>(tile + (8 * j + kr) * 128 + ((part ^ kr) << 4)) = kv[j];
    __builtin_amdgcn_wave_barrier();
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const char* at = tile + (16 * t + i) * 128;
      s[t] = mfma16(*reinterpret_cast<const bf16x8*>(at + ((g ^ (i & 7)) << 4)), q0, f32x4{0.f, 0.f, 0.f, 0.f});
      s[t] = mfma16(*reinterpret_cast<const bf16x8*>(at + (((4 + g) ^ (i & 7)) << 4)), q1, s[t]);
    }
    __builtin_amdgcn_wave_barrier();
    float mx = m;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[t][r] *= c;
        if (base + 64 > k_hi && base + 16 * t + 4 * g + r >= k_hi) s[t][r] = -INFINITY;
        mx = fmaxf(mx, s[t][r]);
      }
    if (W && i < gn) {
      float* dst = a.scores + ((int64_t)b * a.H + h0 + i) * a.score_ld + base + 4 * g;     // (rows are padded to whole batches)
#pragma unroll
      for (int t = 0; t < 4; ++t) *reinterpret_cast<f32x4*>(dst + 16 * t) = s[t];
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float ref = mx == -INFINITY ? 0.f : mx;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mx;
    l *= alpha;
#pragma unroll
    for (int cg = 0; cg < 4; ++cg) acc[cg] *= alpha;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) { s[t][r] = __builtin_amdgcn_exp2f(s[t][r] - ref); l += s[t][r]; }
#pragma unroll
    for (int j = 0; j < 8; ++j) *reinterpret_cast<u32x4*>(tile + (8 * j + kr) * 128 + ((part ^ kr) << 4)) = vv[j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      bf16x8 hi, lo;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = s[2 * u + (j >> 2)][j & 3];
        hi[j] = (__bf16)(p * 0.9961f);                       // 0.9961 (1 + 2^-8) < 1: never rounded up to p, so the rest is over 0
        lo[j] = (__bf16)(p - (float)hi[j]);
      }
#pragma unroll
      for (int cg = 0; cg < 4; ++cg) {
        const int row = 32 * u + 4 * g + (i >> 2), chunk = 2 * cg + ((i & 3) >> 1);
        const char* at = tile + row * 128 + ((chunk ^ (row & 7)) << 4) + (i & 1) * 8;        // (row + 16 has the same row & 7)
        const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(at));
        const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(at + 16 * 128));
        typedef short short8v __attribute__((ext_vector_type(8)));
        const bf16x8 vt = __builtin_bit_cast(bf16x8, (short8v)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        acc[cg] = mfma16(vt, hi, acc[cg]);
        acc[cg] = mfma16(vt, lo, acc[cg]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  // waves -> workgroup, by rescaling with 2^(m - max) in a fixed order.  a wave that met a page outside the pool leaves NaN
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (__any(bad)) l = __builtin_nanf("");
  float* mine = reinterpret_cast<float*>(tile) + i * RED;
#pragma unroll
  for (int cg = 0; cg < 4; ++cg) *reinterpret_cast<f32x4*>(mine + 16 * cg + 4 * g) = acc[cg];
  if (g == 0) { mine[64] = m; mine[65] = l; }
  __syncthreads();
  const bool one = a.nsplit == 1 && !(W && a.nsub > 1);
  float* fin = reinterpret_cast<float*>(lds[0] + HEADS * RED * 4);       // behind the partial results: reference and 1 / sum of the heads
  for (int q = wave; q < gn; q += NW) {
    float mb = -INFINITY, lb = 0.f, ob = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) mb = fmaxf(mb, reinterpret_cast<const float*>(lds[w])[q * RED + 64]);
    const float ref = mb == -INFINITY ? 0.f : mb;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float* part = reinterpret_cast<const float*>(lds[w]) + q * RED;
      const float r = __builtin_amdgcn_exp2f(part[64] - ref);
      lb += part[65] * r;
      ob += part[lane] * r;
    }
    const int h = h0 + q;
    if (one) {
      a.o[b * a.o_s + h * 64 + lane] = f2bf(n_raw == 0 ? 0.f : ob / lb);
      if (W && lane == 0) { fin[q] = ref; fin[HEADS + q] = 1.f / lb; }
    } else {
      float* dst = a.ws + (((int64_t)b * a.H + h) * a.nsplit + split) * PART;
      if (lane == 0) { dst[0] = mb; dst[1] = lb; }
      dst[2 + lane] = ob;
    }
  }
  if (W && one) {                                          // one workgroup has all heads and all keys (nsub is 1): the weights at once
    __syncthreads();
    const float* sc = a.scores + ((int64_t)b * a.H + h0) * a.score_ld;
    float* dst = a.weights + b * a.w_bs + hk * a.w_hs;
    for (int p = threadIdx.x; p < n; p += 64 * NW) {
      float w = 0.f;
#pragma unroll 4
      for (int q = 0; q < gn; ++q) w += __builtin_amdgcn_exp2f(sc[q * a.score_ld + p] - fin[q]) * fin[HEADS + q];
      dst[p] = (has_new && p == n - 1 ? 0.f : dst[p]) + w;
    }
  }
}

// splits of a sequence of length n that hold keys (at least one: split 0 always writes); all of them where the length is outside the table
__device__ __forceinline__ int splits_of(const PagedArgs& a, int n, bool bad) {
  if (bad) return 1;
  const int keys = keys_per_wave(n, a.nw, a.kw_max) * a.nw;
  return max(1, (n + keys - 1) / keys);
}

// maximum (base 2) and sum over the splits of one query head, by one wave; the factor of split lane + 64 j in r[j].  every lane gets the same
__device__ __forceinline__ void join_stats(const float* src, int ns, int lane, float (&r)[MAX_SPLIT / 64], float& mg, float& lg) {
  float ms[MAX_SPLIT / 64], ls[MAX_SPLIT / 64];
  mg = -INFINITY;
#pragma unroll
  for (int j = 0; j < MAX_SPLIT / 64; ++j) {
    const bool in = lane + 64 * j < ns;
    ms[j] = in ? src[(lane + 64 * j) * PART] : -INFINITY;
    ls[j] = in ? src[(lane + 64 * j) * PART + 1] : 0.f;
    mg = fmaxf(mg, ms[j]);
  }
  mg = wave_max(mg);
  const float ref = mg == -INFINITY ? 0.f : mg;
  lg = 0.f;
#pragma unroll
  for (int j = 0; j < MAX_SPLIT / 64; ++j) {
    r[j] = __builtin_amdgcn_exp2f(ms[j] - ref);
    lg += ls[j] * r[j];
  }
  lg = wave_sum(lg);
}

// splits -> output of query head (b, h), by the four waves of a workgroup: a quarter of the splits each, then the quarters in order
__device__ __forceinline__ void join_head(const PagedArgs& a, int b, int h, int n, int ns, float (&fac)[MAX_SPLIT], float (&quarter)[4][64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* src = a.ws + ((int64_t)b * a.H + h) * a.nsplit * PART;
  float r[MAX_SPLIT / 64], mg, lg;
  join_stats(src, ns, lane, r, mg, lg);
  __syncthreads();                                           // (the head before is done with fac and quarter)
  if (wave == 0) {
#pragma unroll
    for (int j = 0; j < MAX_SPLIT / 64; ++j) fac[lane + 64 * j] = r[j];
  }
  __syncthreads();
  float o = 0.f;
#pragma unroll 8
  for (int s = wave; s < ns; s += 4) o = __builtin_fmaf(src[s * PART + 2 + lane], fac[s], o);
  quarter[wave][lane] = o;
  __syncthreads();
  if (wave == 0) {
    o = (quarter[0][lane] + quarter[1][lane]) + (quarter[2][lane] + quarter[3][lane]);
    a.o[b * a.o_s + h * 64 + lane] = f2bf(n == 0 ? 0.f : o / lg);
  }
}

__global__ __launch_bounds__(256) void paged_join_kernel(const PagedArgs a) {
  __shared__ float fac[MAX_SPLIT], quarter[4][64];
  const int b = blockIdx.x / a.H, n = a.lengths[b];
  const bool bad = n < 0 || n > a.pg.cap;
  join_head(a, b, blockIdx.x % a.H, n, splits_of(a, n, bad), fac, quarter);
}

// splits -> outputs and scores -> weights: a workgroup per key-value head and 1024 positions adds the weights of its heads there; the workgroups
// behind those join the outputs, one query head each.  Reads the scores that the attending launch has left in the caches: 128 heads of 6189 keys 5.5 us,
// of 24935 18 us (1024 positions: 512, 2048 and 4096 were no faster).  A workgroup of its own per output head costs nothing beside that.
__global__ __launch_bounds__(256) void paged_join_weights_kernel(const PagedArgs a, int wblocks) {
  __shared__ float fac[MAX_SPLIT], quarter[4][64], ref[HEADS], inv[HEADS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x / a.Hkv, hk = blockIdx.x % a.Hkv;
  const int h0 = hk * a.group;
  const int n = a.lengths[b];
  const bool bad = n < 0 || n > a.pg.cap;
  const int ns = splits_of(a, n, bad);
  if ((int)blockIdx.y >= wblocks) {
    join_head(a, b, h0 + blockIdx.y - wblocks, n, ns, fac, quarter);
    return;
  }
  const int p0 = blockIdx.y * 1024 + threadIdx.x;
  if (bad || (int)blockIdx.y * 1024 >= n) return;
  float* dst = a.weights + b * a.w_bs + hk * a.w_hs;
  float w[4], old[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = p0 + i * 256;
    old[i] = p < n && !(a.k_new && p == n - 1) ? dst[p] : 0.f;
    w[i] = 0.f;
  }
  for (int g0 = 0; g0 < a.group; g0 += HEADS) {
    const int gn = min(HEADS, a.group - g0);
    if (g0) __syncthreads();
    for (int g = wave; g < gn; g += 4) {
      float r[MAX_SPLIT / 64], mg, lg;
      join_stats(a.ws + ((int64_t)b * a.H + h0 + g0 + g) * a.nsplit * PART, ns, lane, r, mg, lg);
      if (lane == 0) { ref[g] = mg == -INFINITY ? 0.f : mg; inv[g] = 1.f / lg; }
    }
    __syncthreads();
    const float* sc = a.scores + ((int64_t)b * a.H + h0 + g0) * a.score_ld;
#pragma unroll 4
    for (int g = 0; g < gn; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = min(p0 + i * 256, n - 1);
        w[i] += __builtin_amdgcn_exp2f(sc[g * a.score_ld + p] - ref[g]) * inv[g];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = p0 + i * 256;
    if (p < n) dst[p] = old[i] + w[i];
  }
}

// rows [b, t] -> position starts[b] + t, t < counts[b]; 16 bytes a thread, all loads independent.  64 rows of 16 sequences, 16 heads, 8.4 MB read
// and written: 4 to 5 us, little over an empty launch
__global__ __launch_bounds__(256) void paged_append_kernel(const u16* k, const u16* v, int64_t k_bs, int64_t k_rs, int64_t v_bs, int64_t v_rs,
                                                           u16* kp, u16* vp, const Pages pg, const int* starts, const int* counts,
                                                           float* weights, int64_t w_bs, int64_t w_hs, int T, int Hkv) {
  const int b = blockIdx.y;
  const int count = min(counts[b], T), start = starts[b];
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int t = (int)(i / (Hkv * 8)), r = (int)(i % (Hkv * 8)), h = r >> 3, part = r & 7;
  if (t >= count || start > pg.cap - 1 - t || start < -t) return;        // (no sum that could pass 32 bits)
  const int p = start + t;
  int64_t to;
  if (!row_of(pg, pg.table + b * pg.table_ld, p, to)) return;
  to += h * pg.head_s + 8 * part;
  *reinterpret_cast<uint4*>(kp + to) = *reinterpret_cast<const uint4*>(k + b * k_bs + t * k_rs + 8 * r);
  *reinterpret_cast<uint4*>(vp + to) = *reinterpret_cast<const uint4*>(v + b * v_bs + t * v_rs + 8 * r);
  if (weights && part == 0) weights[b * w_bs + h * w_hs + p] = 0.f;
}

// one token per sequence, each at a position of its own: a wave per row.  ids or positions outside their tables: NaN rows, nothing is read
__global__ __launch_bounds__(256) void embed_rows_kernel(const int64_t* ids, const float* tok, const float* pos, float* out, int B, int D, int off,
                                                         int vocab, const int* positions, int n_pos) {
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= B) return;
  const int64_t id = ids[row], p = (int64_t)positions[row] + off;
  const bool ok = id >= 0 && id < vocab && p >= 0 && p < n_pos;
  for (int c = lane * 4; c < D; c += 256) {
    f32x4 x;
    if (ok) x = *reinterpret_cast<const f32x4*>(tok + id * D + c) + *reinterpret_cast<const f32x4*>(pos + p * D + c);
    else x = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
    *reinterpret_cast<f32x4*>(out + (int64_t)row * D + c) = x;
  }
}

// ------------------------------------------------------------------------------------------------------------- eviction
struct EvictArgs {
  u16 *k, *v;
  Pages pg;
  const int* lengths;
  int* new_lengths;
  float* weights; int64_t w_bs, w_hs;
  int* kept;                            // [B * Hkv][budget]
  int* moved;                           // [B * Hkv] rows that the second launch moves: budget, or 0 for a sequence that stays as it is
  int B, Hkv, budget, recent;
};

// a whole number in the order of the float: NaN above all, -0 with +0
__device__ __forceinline__ uint32_t order_key(float x) {
  if (!(x == x)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int SEL = 1024, SK = 8;       // threads of the selecting workgroup, positions of a thread: 8192 of a sequence at once
constexpr int RB = 11, RN = 1 << RB;    // radix digits of 11, 11 and 10 bits

// inclusive sums over the lanes of a wave on the DPP path
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t add_shifted(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {
  v = add_shifted<0x111, 0xf>(v);
  v = add_shifted<0x112, 0xf>(v);
  v = add_shifted<0x114, 0xf>(v);
  v = add_shifted<0x118, 0xf>(v);
  v = add_shifted<0x142, 0xa>(v);
  return add_shifted<0x143, 0xc>(v);
}
// exclusive sums over the workgroup (one barrier; `sh` may be used again after the next one), and the total
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t* sh, uint32_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t incl = wave_prefix(v);
  if (lane == 63) sh[wave] = incl;
  __syncthreads();
  uint32_t before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < SEL / 64; ++w) { const uint32_t x = sh[w]; before += w < wave ? x : 0; all += x; }
  return before + incl - v;
}

// Rows of one pool move down in place, by a workgroup of 1024 threads that walks the kept list in tiles of 1024, in order.  Row i comes from
// position kept[i] >= i, so a tile's rows are all read before any of it is written (barrier), and no tile reads what an earlier one wrote: the
// next tile's rows are on their way while this one's are stored.  Bound by the rows, read and written once: 128 heads
// that keep 2048 of 6189, 134 MB in 23.7 us, 5.7 TB/s.
// LPR: lanes a row, 16 bytes each: 8 move it whole, fewer a slice of it, which other workgroups complete.
constexpr int MU = 8, MTILE = SEL / 8 * MU;                // instructions a tile, rows of a tile of whole rows
template <int LPR>
__device__ __forceinline__ void move_rows(const Pages& pg, const int* table, u16* rows, const int* kept, int count) {
  constexpr int MROWS = SEL / LPR, MTILE = MROWS * MU;     // rows per load instruction of the workgroup, rows per tile
  const int row = threadIdx.x / LPR;
  u16* base = rows + 8 * (threadIdx.x % LPR);
  u32x4 x[2][MU];
  uint32_t ok[2];
  const auto load = [&](int t0, u32x4 (&v)[MU], uint32_t& good) {
    good = 0;
#pragma unroll
    for (int j = 0; j < MU; ++j) {
      const int i = t0 + j * MROWS + row;
      int64_t from;
      if (row_of(pg, table, kept[min(i, count - 1)], from) && i < count) good |= 1u << j;
      v[j] = *reinterpret_cast<const u32x4*>(base + from);
    }
  };
  const auto store = [&](int t0, u32x4 (&v)[MU], uint32_t good) {
#pragma unroll
    for (int j = 0; j < MU; ++j) asm volatile("" : "+v"(v[j]));          // this tile's rows have arrived (the next one's have not)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < MU; ++j) {
      int64_t to;
      if ((good >> j & 1) && row_of(pg, table, t0 + j * MROWS + row, to)) *reinterpret_cast<u32x4*>(base + to) = v[j];
    }
  };
  load(0, x[0], ok[0]);
  for (int t0 = 0; t0 < count; t0 += 2 * MTILE) {
    if (t0 + MTILE < count) load(t0 + MTILE, x[1], ok[1]);
    store(t0, x[0], ok[0]);
    if (t0 + MTILE < count) {
      if (t0 + 2 * MTILE < count) load(t0 + 2 * MTILE, x[0], ok[0]);
      store(t0 + MTILE, x[1], ok[1]);
    }
  }
}

// the same for up to one tile of rows of both pools, K and V under way together
__device__ __forceinline__ void move_tile(const Pages& pg, const int* table, u16* k, u16* v, const uint32_t* kept, int count) {
  constexpr int MROWS = SEL / 8;
  const int row = threadIdx.x >> 3, part = 8 * (threadIdx.x & 7);
  u32x4 x[2][MU];
  uint32_t good = 0;
#pragma unroll
  for (int j = 0; j < MU; ++j) {
    const int i = j * MROWS + row;
    int64_t from;
    if (row_of(pg, table, (int)kept[min(i, count - 1)], from) && i < count) good |= 1u << j;
    x[0][j] = *reinterpret_cast<const u32x4*>(k + part + from);
    x[1][j] = *reinterpret_cast<const u32x4*>(v + part + from);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < MU; ++j) {
    int64_t to;
    if (!(good >> j & 1) || !row_of(pg, table, j * MROWS + row, to)) continue;
    *reinterpret_cast<u32x4*>(k + part + to) = x[0][j];
    *reinterpret_cast<u32x4*>(v + part + to) = x[1][j];
  }
}

// One workgroup per (sequence, key-value head).  The `need`-th largest weight among the old positions by a radix selection (digits of 11, 11
// and 10 bits, histogram in LDS), then one ordered pass that writes the kept positions and moves their weights down.  A thread holds up to 8
// neighbouring positions in registers; a sequence of up to 8192 is read once.  Integer atomics only: the result does not depend on their order.
// The page ids are looked over while the weights are on their way, in the barrier that the empty histogram needs anyway: 0.2 us of 17 for 256 heads.
// MOVE: the same workgroup then moves the rows of K and V.  Bound by the rounds of the selection (read, three histograms, the ordered pass; each waits
// for the one before): 11.5 us for 128 heads of 6189 positions, whose 3.2 MB take under 1; with MOVE, 96 heads of 1023 that keep 512, 13.4 us.
template <bool MOVE>
__global__ __launch_bounds__(SEL) void evict_select_kernel(const EvictArgs a) {
  __shared__ uint32_t hist[RN];
  __shared__ uint32_t sh[2][SEL / 64];
  __shared__ uint32_t pick[2];
  const int tid = threadIdx.x;
  const int bh = blockIdx.x, b = bh / a.Hkv, h = bh % a.Hkv;
  const int n = a.lengths[b];
  int* kept = a.kept + (int64_t)bh * a.budget;
  const int* table = a.pg.table + b * a.pg.table_ld;
  const auto leave = [&](int stay) {    // the sequence as it is; of the list, its first `stay` positions
    if (MOVE && h == 0 && tid == 0) a.new_lengths[b] = n;
    if (!MOVE && tid == 0) a.moved[bh] = 0;
    for (int i = tid; i < a.budget; i += SEL) kept[i] = i < stay ? i : -1;
  };
  if (n < 0 || n > a.pg.cap || n <= a.budget) { leave(n > a.pg.cap ? 0 : n); return; }
  float* w = a.weights + b * a.w_bs + h * a.w_hs;
  const int old = n - a.recent;         // recent <= budget < n
  uint32_t need = a.budget - a.recent;  // how many of the old ones stay
  const bool some = need > 0;
  uint32_t prefix = 0, mask = 0;        // the digits of the threshold found so far
  const int per = min(SK, (n + SEL - 1) / SEL), tile = SEL * per;        // short sequences are spread over the threads too
  float x[SK];
  const auto load = [&](int t0) {
#pragma unroll
    for (int k = 0; k < SK; ++k)
      if (k < per) x[k] = w[min(t0 + tid * per + k, n - 1)];
  };
  const bool once = n <= tile;
  if (once) load(0);
  // one page outside the pool leaves the whole sequence as it is: every head of it looks at the same entries and finds the same
  bool off = false;
  for (int i = tid; i <= (n - 1) >> a.pg.shift; i += SEL) off |= (unsigned)table[i] >= (unsigned)a.pg.n_pages;
  const bool off_wave = __any(off);
  if ((tid & 63) == 0) sh[1][tid >> 6] = off_wave;
  for (int i = tid; i < RN; i += SEL) hist[i] = 0;
  __syncthreads();
  uint32_t off_any = 0;
#pragma unroll
  for (int i = 0; i < SEL / 64; ++i) off_any |= sh[1][i];
  if (off_any) { leave(0); return; }
  if (MOVE && h == 0 && tid == 0) a.new_lengths[b] = a.budget;
  if (!MOVE && tid == 0) a.moved[bh] = a.budget;
  if (some) {
    for (int pass = 0; pass < 3; ++pass) {
      const int sft = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t bins = pass == 2 ? 1 << 10 : RN;
      for (int t0 = 0; t0 < old; t0 += tile) {
        if (!once) load(t0);
#pragma unroll
        for (int k = 0; k < SK; ++k) {
          if (k >= per) break;
          const uint32_t u = order_key(x[k]);
          if (t0 + tid * per + k < old && (u & mask) == prefix) atomicAdd(&hist[(u >> sft) & (bins - 1)], 1u);
        }
      }
      __syncthreads();
      // the bin in which the need-th largest lies: thread t takes the t-th two bins from the top, and leaves them empty
      const int hi = RN - 1 - 2 * tid;
      const uint32_t c0 = hist[hi], c1 = hist[hi - 1];
      hist[hi] = hist[hi - 1] = 0;
      uint32_t all;
      const uint32_t above = block_prefix(c0 + c1, sh[0], all);
      if (above < need && need <= above + c0) { pick[0] = hi; pick[1] = above; }
      else if (above + c0 < need && need <= above + c0 + c1) { pick[0] = hi - 1; pick[1] = above + c0; }
      __syncthreads();
      prefix |= pick[0] << sft;
      mask |= (bins - 1) << sft;
      need -= pick[1];
    }
  }
  // kept: above the threshold or recent ("sure"), or equal to it and among the first `need` of the equal ones
  uint32_t sure_out = 0, tie_out = 0;
  for (int t0 = 0, side = 0; t0 < n; t0 += tile, side ^= 1) {
    if (!once) load(t0);
    uint32_t sure = 0, tie = 0;         // bits
#pragma unroll
    for (int k = 0; k < SK; ++k) {
      if (k >= per) break;
      const int p = t0 + tid * per + k;
      const uint32_t u = order_key(x[k]);
      if (p >= old ? p < n : some && u > prefix) sure |= 1u << k;
      if (p < old && some && u == prefix) tie |= 1u << k;
    }
    uint32_t all;                       // (the barrier also orders every read of this tile before the writes below; counts of 16 bits each)
    const uint32_t at = block_prefix((uint32_t)__popc(sure) << 16 | __popc(tie), sh[side], all);
    uint32_t sb = sure_out + (at >> 16), tb = tie_out + (at & 0xffff);
#pragma unroll
    for (int k = 0; k < SK; ++k) {
      const bool is_sure = sure >> k & 1, is_tie = tie >> k & 1;
      if (is_sure || (is_tie && tb < need)) {
        const uint32_t to = sb + min(tb, need);
        kept[to] = t0 + tid * per + k;
        if (MOVE && to < MTILE) hist[to] = t0 + tid * per + k;             // (the histogram has done its work)
        w[to] = x[k];
      }
      sb += is_sure;
      tb += is_tie;
    }
    sure_out += all >> 16;
    tie_out += all & 0xffff;
  }
  if (MOVE) {
    __syncthreads();                    // the list is complete
    u16 *k = a.k + h * a.pg.head_s, *v = a.v + h * a.pg.head_s;
    if (a.budget <= MTILE) {
      move_tile(a.pg, table, k, v, hist, a.budget);
    } else {
      move_rows<8>(a.pg, table, k, kept, a.budget);
      move_rows<8>(a.pg, table, v, kept, a.budget);
    }
  }
}

// the rows of one (sequence, head), K or V, or slices of them
template <int LPR>
__global__ __launch_bounds__(SEL) void evict_move_kernel(const EvictArgs a) {
  const int bh = blockIdx.x, b = bh / a.Hkv, h = bh % a.Hkv;
  const int count = a.moved[bh];
  if (h == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.new_lengths[b] = count ? count : a.lengths[b];
  if (count == 0) return;
  move_rows<LPR>(a.pg, a.pg.table + b * a.pg.table_ld, (blockIdx.y & 1 ? a.v : a.k) + h * a.pg.head_s + 8 * LPR * (blockIdx.y >> 1),
                 a.kept + (int64_t)bh * a.budget, count);
}

int log2_of(int x) { int s = 0; while ((1 << s) < x) ++s; return s; }

// checks what the four entry points share about a pool; 0 or -1
int check_pool(const char* who, const void* k, const void* v, int64_t page_s, int64_t row_s, int64_t head_s, int n_pages, int page_size,
               const int* table, int64_t table_ld, int max_pages, int B, int Hkv) {
  CRL_CHECK(k && v && table, "%s: null pointer", who);
  CRL_CHECK(B > 0 && Hkv > 0 && n_pages > 0 && max_pages > 0, "%s: empty problem", who);
  CRL_CHECK(page_size >= 1 && page_size <= 4096 && (page_size & (page_size - 1)) == 0, "%s: page_size %d is not a power of two up to 4096", who, page_size);
  CRL_CHECK((int64_t)max_pages * page_size < (1ll << 30), "%s: a sequence's table covers 2^30 positions or more", who);
  CRL_CHECK(table_ld >= max_pages, "%s: page table rows overlap", who);
  CRL_CHECK(((uintptr_t)k % 16) == 0 && ((uintptr_t)v % 16) == 0 && (page_s % 8) == 0 && (row_s % 8) == 0 && (head_s % 8) == 0,
            "%s: pages must be 16-byte aligned with strides multiple of 8 elements", who);
  return 0;
}

Pages pages_of(const int* table, int64_t table_ld, int64_t page_s, int64_t row_s, int64_t head_s, int n_pages, int page_size, int max_pages) {
  return Pages{table, table_ld, page_s, row_s, head_s, n_pages, log2_of(page_size), max_pages * page_size};
}

// Splits of a sequence's capacity.  One (no joining launch, 3 to 4 us) where eight waves get through it in two or four batches each; with weights
// only if the workgroup has all query heads and few scores to go over again.  Else 2048 workgroups, twice what is resident, of 256 keys or more.
// One split against several, full sequences, in us:
//   capacity                                512          1024          2048          4096
//   12 workgroups                        5.3 / 7.6     7.6 / 7.7    12.2 / 8.3    20.9 / 9.7
//   64 workgroups                        5.6 / 8.1     7.8 / 9.4    14.6 / 13.1   25.0 / 19.2
//   256 workgroups                       9.3 / 12.7   14.7 / 18.4   26.6 / 30.6   49.1 / 53.4
//   12 heads, weights                    6.6 / 8.6     9.7 / 9.0    15.8 / 9.2    27.0 / 9.9
//   16 heads on 4 (32 wg), weights       7.3 / 9.0    10.2 / 9.5    16.4 / 10.6   34.4 / 14.6
//   256 heads, weights                  11.1 / 13.9   18.4 / 21.3   33.3 / 34.1   61.6 / 62.8
// The rule is on the right side but for 12 to 64 workgroups at its border (up to 1.5 us).
int paged_plan(int blocks, int nsub, int group, int cap, bool weights) {
  if (cap <= (blocks >= 64 ? 2048 : 1024) && !(weights && (nsub > 1 || (int64_t)cap * group > W_DIRECT))) return 1;
  const int max_split = (cap + 255) / 256;
  int ns = (2048 + blocks - 1) / blocks;
  ns = ns < 1 ? 1 : (ns > max_split ? max_split : ns);
  return ns > MAX_SPLIT ? MAX_SPLIT : ns;
}

int64_t score_row(int cap) { return ((int64_t)cap + 63) / 64 * 64; }

}  // namespace

extern "C" int crl_paged_row(const int* host_table_row, int position, int64_t page_s, int64_t row_s, int n_pages, int page_size, int max_pages,
                             int64_t* offset) {
  CRL_CHECK(host_table_row && offset && n_pages > 0 && page_size >= 1 && page_size <= 4096 && (page_size & (page_size - 1)) == 0 && max_pages >= 1,
            "crl_paged_row: bad arguments");
  if (position < 0 || position / page_size >= max_pages) return 1;
  return row_of(pages_of(nullptr, 0, page_s, row_s, 0, n_pages, page_size, max_pages), host_table_row, position, *offset) ? 0 : 1;
}

extern "C" size_t crl_paged_attn_decode_ws_bytes(int B, int H, int Hkv, int page_size, int max_pages, int with_weights) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || page_size <= 0 || max_pages <= 0 || (int64_t)page_size * max_pages > INT_MAX) return 0;
  const int nsub = (H / Hkv + HEADS - 1) / HEADS, cap = page_size * max_pages;
  const int nsplit = paged_plan(B * Hkv * nsub, nsub, H / Hkv, cap, with_weights != 0);
  if (nsplit == 1 && !with_weights) return 0;
  size_t bytes = (size_t)B * H * nsplit * PART * sizeof(float);
  bytes = (bytes + 255) / 256 * 256;
  if (with_weights) bytes += (size_t)B * H * score_row(cap) * sizeof(float);
  return bytes;
}

extern "C" int crl_paged_attn_decode(const void* q, int64_t q_s, void* k_pages, void* v_pages, int64_t page_s, int64_t row_s, int64_t head_s,
                                     int n_pages, int page_size, const int* page_table, int64_t table_ld, int max_pages, const int* lengths,
                                     const void* k_new, int64_t k_new_s, const void* v_new, int64_t v_new_s, void* o, int64_t o_s,
                                     float* weights, int64_t w_bs, int64_t w_hs, int B, int H, int Hkv, float scale, void* ws, size_t ws_bytes,
                                     void* stream) {
  const char* who = "crl_paged_attn_decode";
  CRL_CHECK(q && o && lengths, "%s: null pointer", who);
  if (int rc = check_pool(who, k_pages, v_pages, page_s, row_s, head_s, n_pages, page_size, page_table, table_ld, max_pages, B, Hkv)) return rc;
  CRL_CHECK(H > 0 && H % Hkv == 0, "%s: %d query heads over %d key-value heads", who, H, Hkv);
  CRL_CHECK((k_new != nullptr) == (v_new != nullptr), "%s: k_new and v_new go together", who);
  CRL_CHECK(((uintptr_t)q % 16) == 0 && (q_s % 8) == 0 && ((uintptr_t)k_new % 16) == 0 && ((uintptr_t)v_new % 16) == 0 && (k_new_s % 8) == 0 &&
                (v_new_s % 8) == 0, "%s: q, k_new and v_new must be 16-byte aligned with strides multiple of 8 elements", who);
  PagedArgs a{};
  a.q = (const u16*)q; a.k_new = (const u16*)k_new; a.v_new = (const u16*)v_new; a.k = (u16*)k_pages; a.v = (u16*)v_pages; a.o = (u16*)o;
  a.q_s = q_s; a.o_s = o_s; a.kn_s = k_new_s; a.vn_s = v_new_s;
  a.pg = pages_of(page_table, table_ld, page_s, row_s, head_s, n_pages, page_size, max_pages);
  a.lengths = lengths; a.weights = weights; a.w_bs = w_bs; a.w_hs = w_hs;
  a.B = B; a.H = H; a.Hkv = Hkv; a.group = H / Hkv; a.nsub = (a.group + HEADS - 1) / HEADS; a.scale = scale;
  CRL_CHECK((int64_t)B * Hkv * a.nsub < (1ll << 31) && (int64_t)B * H < (1ll << 31), "%s: too many sequences", who);
  a.nsplit = paged_plan(B * Hkv * a.nsub, a.nsub, a.group, a.pg.cap, weights != nullptr);
  const bool join_weights = weights && (a.nsplit > 1 || a.nsub > 1);
  const int wblocks = (a.pg.cap + 1023) / 1024;              // 1024 positions each of the joining launch
  CRL_CHECK(!join_weights || wblocks + a.group < 65536, "%s: weights of %d positions and %d query heads a key-value head are too many", who, a.pg.cap, a.group);
  const size_t want = crl_paged_attn_decode_ws_bytes(B, H, Hkv, page_size, max_pages, weights != nullptr);
  CRL_CHECK(want == 0 || (ws && ws_bytes >= want), "%s: workspace too small (%zu bytes, %zu needed)", who, ws_bytes, want);
  a.ws = (float*)ws;
  a.score_ld = score_row(a.pg.cap);
  a.scores = weights ? (float*)((char*)ws + (want - (size_t)B * H * a.score_ld * sizeof(float))) : nullptr;
  hipStream_t s = as_stream(stream);
  const dim3 grid((unsigned)(B * Hkv * a.nsub), (unsigned)a.nsplit);
  // Workgroups go to the eight XCDs in turn, so without this a head would be one XCD's in every split: long sequences of a ragged batch would pile up
  // there, and where the rows of a head are not next to each other all that an XCD reads would come through a few of its L2 channels.  Ragged, 16
  // heads on 4: 26.8 us against 29.4; 24935 keys, 16 heads, rows of all heads together: 152 against 166 (rows of a head together: 150 either way).  With
  // weights, the joining launch finds a head's scores in the L2 of the XCD that wrote them: 48.3 against 48.9, and 50.2 against 53.9 for rows of
  // all heads together.
  a.turn = !weights || row_s > 64 ? 3 : 0;
  const bool wide = a.nsplit == 1 && a.pg.cap > 256 && grid.x < 1024;
  a.nw = wide ? 8 : 4;
  a.kw_max = ((a.pg.cap + a.nsplit * a.nw - 1) / (a.nsplit * a.nw) + 63) & ~63;
  if (wide) { if (weights) paged_attn_kernel<8, true><<<grid, 512, 0, s>>>(a); else paged_attn_kernel<8, false><<<grid, 512, 0, s>>>(a); }
  else { if (weights) paged_attn_kernel<4, true><<<grid, 256, 0, s>>>(a); else paged_attn_kernel<4, false><<<grid, 256, 0, s>>>(a); }
  CRL_LAUNCH_CHECK(who);
  if (join_weights) {
    paged_join_weights_kernel<<<dim3((unsigned)(B * Hkv), (unsigned)(wblocks + a.group)), 256, 0, s>>>(a, wblocks);
    CRL_LAUNCH_CHECK("crl_paged_attn_decode(join, weights)");
  } else if (a.nsplit > 1) {
    paged_join_kernel<<<(unsigned)(B * H), 256, 0, s>>>(a);
    CRL_LAUNCH_CHECK("crl_paged_attn_decode(join)");
  }
  return 0;
}

extern "C" int crl_paged_append(const void* k, int64_t k_bs, int64_t k_rs, const void* v, int64_t v_bs, int64_t v_rs, void* k_pages, void* v_pages,
                                int64_t page_s, int64_t row_s, int64_t head_s, int n_pages, int page_size, const int* page_table, int64_t table_ld,
                                int max_pages, const int* starts, const int* counts, float* weights, int64_t w_bs, int64_t w_hs, int B, int T,
                                int Hkv, void* stream) {
  const char* who = "crl_paged_append";
  CRL_CHECK(k && v && starts && counts, "%s: null pointer", who);
  if (int rc = check_pool(who, k_pages, v_pages, page_s, row_s, head_s, n_pages, page_size, page_table, table_ld, max_pages, B, Hkv)) return rc;
  CRL_CHECK(T > 0 && (int64_t)T * Hkv * 8 < (1ll << 38) && B < 65536, "%s: bad shape B=%d T=%d", who, B, T);
  CRL_CHECK(((uintptr_t)k % 16) == 0 && ((uintptr_t)v % 16) == 0 && (k_bs % 8) == 0 && (k_rs % 8) == 0 && (v_bs % 8) == 0 && (v_rs % 8) == 0,
            "%s: rows must be 16-byte aligned with strides multiple of 8 elements", who);
  const Pages pg = pages_of(page_table, table_ld, page_s, row_s, head_s, n_pages, page_size, max_pages);
  const dim3 grid((unsigned)(((int64_t)T * Hkv * 8 + 255) / 256), (unsigned)B);
  paged_append_kernel<<<grid, 256, 0, as_stream(stream)>>>((const u16*)k, (const u16*)v, k_bs, k_rs, v_bs, v_rs, (u16*)k_pages, (u16*)v_pages, pg,
                                                           starts, counts, weights, w_bs, w_hs, T, Hkv);
  CRL_LAUNCH_CHECK(who);
  return 0;
}

extern "C" size_t crl_cache_evict_ws_bytes(int B, int Hkv, int budget) {
  if (B <= 0 || Hkv <= 0 || budget < 0) return 0;
  return (size_t)B * Hkv * sizeof(int) * ((size_t)budget + 1);
}

extern "C" int crl_cache_evict(void* k_pages, void* v_pages, int64_t page_s, int64_t row_s, int64_t head_s, int n_pages, int page_size,
                               const int* page_table, int64_t table_ld, int max_pages, const int* lengths, float* weights, int64_t w_bs,
                               int64_t w_hs, int B, int Hkv, int budget, int recent, int* new_lengths, int* kept, void* ws, size_t ws_bytes,
                               void* stream) {
  const char* who = "crl_cache_evict";
  CRL_CHECK(lengths && weights && new_lengths && ws, "%s: null pointer", who);
  if (int rc = check_pool(who, k_pages, v_pages, page_s, row_s, head_s, n_pages, page_size, page_table, table_ld, max_pages, B, Hkv)) return rc;
  CRL_CHECK(budget > 0 && recent >= 0 && recent <= budget, "%s: budget %d, recent %d", who, budget, recent);
  CRL_CHECK((int64_t)B * Hkv < (1ll << 31), "%s: too many sequences", who);
  CRL_CHECK(ws_bytes >= crl_cache_evict_ws_bytes(B, Hkv, kept ? 0 : budget), "%s: workspace too small (%zu bytes)", who, ws_bytes);
  EvictArgs a{};
  a.k = (u16*)k_pages; a.v = (u16*)v_pages;
  a.pg = pages_of(page_table, table_ld, page_s, row_s, head_s, n_pages, page_size, max_pages);
  a.lengths = lengths; a.new_lengths = new_lengths; a.weights = weights; a.w_bs = w_bs; a.w_hs = w_hs;
  a.moved = (int*)ws;
  a.kept = kept ? kept : (int*)ws + (int64_t)B * Hkv;
  a.B = B; a.Hkv = Hkv; a.budget = budget; a.recent = recent;
  hipStream_t s = as_stream(stream);
  // One launch where a workgroup a head is enough for the rows too: few of them, or heads for every CU.  The lengths must not change under the
  // other heads of a sequence, so not in place.  One launch against two on the GPU (the second costs the host 4 us), half of the positions kept, in us:
  //   rows kept          512          1024          2048
  //   16 heads       11.1 / 11.2   14.0 / 13.0   26.7 / 17.5
  //   128 heads      14.2 / 15.2   21.0 / 20.7   45.0 / 43.1
  //   256 heads      18.6 / 23.7   39.0 / 42.4   76.1 / 77.8
  //   512 heads      44.9 / 47.2   74.9 / 77.8   135.7 / 140.6
  const bool apart = (const char*)new_lengths + 4ll * B <= (const char*)lengths || (const char*)lengths + 4ll * B <= (const char*)new_lengths;
  if (apart && (budget <= MTILE || B * Hkv >= 256)) {
    evict_select_kernel<true><<<(unsigned)(B * Hkv), SEL, 0, s>>>(a);
    CRL_LAUNCH_CHECK(who);
  } else {
    evict_select_kernel<false><<<(unsigned)(B * Hkv), SEL, 0, s>>>(a);
    CRL_LAUNCH_CHECK("crl_cache_evict(select)");
    // A workgroup must take all rows of what it moves, in order, so few heads leave CUs idle: then a row is moved in slices, by two or four
    // workgroups.  In us with whole rows, halves, quarters: 16 heads that keep 9000 rows of 12000 75 / 62 / 59 (32 heads, 6091 of 10247: 62 / 54 / 54);
    // 64 heads, 3000 of 6189: 33 / 28 / 38; 96 heads: 41 / 48 / 70.  With 256 workgroups there, half and quarter cache lines cost
    // more than further CUs bring.
    if (B * Hkv <= 32) evict_move_kernel<2><<<dim3((unsigned)(B * Hkv), 8), SEL, 0, s>>>(a);
    else if (B * Hkv <= 64) evict_move_kernel<4><<<dim3((unsigned)(B * Hkv), 4), SEL, 0, s>>>(a);
    else evict_move_kernel<8><<<dim3((unsigned)(B * Hkv), 2), SEL, 0, s>>>(a);
    CRL_LAUNCH_CHECK("crl_cache_evict(move)");
  }
  return 0;
}

extern "C" int crl_embed_decode_rows(const int64_t* ids, const float* tok, const float* pos, float* out, int B, int D, int pos_offset, int vocab,
                                     const int* positions, int n_pos, void* stream) {
  CRL_CHECK(ids && tok && pos && out && positions, "crl_embed_decode_rows: null pointer");
  CRL_CHECK(B > 0 && D > 0 && (D % 4) == 0 && vocab > 0 && n_pos > 0, "crl_embed_decode_rows: bad shape");
  CRL_CHECK(((uintptr_t)tok % 16) == 0 && ((uintptr_t)pos % 16) == 0 && ((uintptr_t)out % 16) == 0, "crl_embed_decode_rows: 16-byte alignment required");
  embed_rows_kernel<<<(unsigned)((B + 3) / 4), 256, 0, as_stream(stream)>>>(ids, tok, pos, out, B, D, pos_offset, vocab, positions, n_pos);
  CRL_LAUNCH_CHECK("crl_embed_decode_rows");
  return 0;
}
