// fa_cache_append.cu -- new keys and values into the pages of an 8-bit cache, with the position
// rotation of k (and of q) on the way.  No counterpart in the reference, which has no cache.
//
// For the new token at position p of its sequence and a head row x[D], the rotation over the first
// r = rot_dim elements is, for the pairs (a, b) = (x[j], x[j + r/2]) (or (x[2j], x[2j+1]) when
// interleaved) and c = cos[p][j], s = sin[p][j]:  a' = a c - b s,  b' = b c + a s.
//
// A page of one kv head has one scale 2^e for its keys and one for its values.  With A the largest
// finite magnitude among the rows that a call adds to the page, the page needs the least e in
// [-64, 120] with A <= 448 * 2^e; a page that already holds earlier rows keeps the larger of that
// and its own exponent, and where it grows the earlier rows are rounded once more to the new step.
// Scales are powers of two, so dividing by them is exact: the only rounding is the one to e4m3.
//
// The rotation a c + b s is computed as an unevaluated sum of two floats, two sums at a time: both
// products exactly (their rounding errors by fma), the sum's rounding error by the two-sum of Knuth.
// What is stored or returned is then the rounding of the exact value, whatever the order of
// operations.  For k, which is rounded once its page's scale is known, the sum is rounded to odd in 32
// bits (the last bit set where it is inexact): a later rounding to 8 bits is that of the exact value.
// For q the first float, which is the exact value rounded, is rounded again at once; that differs only
// where it lies halfway between two 16-bit values, one in 2^13 or 2^16, and those are done over by way
// of the rounding to odd.  In 64-bit arithmetic the conversions, 16 a cycle, took 129 us for 13613
// tokens of 32 + 8 + 8 heads of 128, and one sum at a time with every one rounded to odd 136 us; the
// memory needs 47.
#include <algorithm>
#include <cmath>

#include "fa_cache_common.cuh"
#include "sm100_ptx.cuh"

namespace fa_sm100 {
namespace {

constexpr int kMinExp = -64;
constexpr int kMaxExp = 120;

__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }

constexpr uint64_t kMinusOne2 = 0xbf800000bf800000ull;

// a c + b s for two lanes of a packed pair: the nearest floats, and in `lo` what is left.
struct Sum2 {
  uint64_t hi, lo;
};
__device__ __forceinline__ Sum2 sum2(uint64_t a, uint64_t c, uint64_t b, uint64_t s) {
  const uint64_t p = f2_mul(a, c), q = f2_mul(b, s);
  const uint64_t minus_p = f2_mul(p, kMinusOne2);
  const uint64_t pe = f2_fma(a, c, minus_p);                      // exact
  const uint64_t qe = f2_fma(b, s, f2_mul(q, kMinusOne2));        // exact
  const uint64_t d = f2_add(p, q);
  const uint64_t t = f2_add(d, minus_p);
  const uint64_t de = f2_add(f2_fma(f2_fma(t, kMinusOne2, d), kMinusOne2, p),
                             f2_fma(t, kMinusOne2, q));           // p + q = d + de
  const uint64_t e = f2_add(de, f2_add(pe, qe));
  const uint64_t h = f2_add(d, e);
  return Sum2{h, f2_fma(f2_fma(d, kMinusOne2, h), kMinusOne2, e)};
}

// h + lo rounded to odd; where h is not finite because of the steps above, `plain` is the value.
__device__ __forceinline__ float to_odd(float h, float lo, float plain) {
  const int bits = __float_as_int(h);
  if (!(fabsf(h) < INFINITY)) return plain;
  // The value lies between h and its neighbour on lo's side; one of the two is odd.
  const int toward = (__float_as_int(lo) ^ bits) < 0 ? -1 : 1;
  return lo != 0.f && (bits & 1) == 0 ? __int_as_float(bits + toward) : h;
}

__device__ __forceinline__ float finite_or_nan(float x) {
  return fabsf(x) < INFINITY ? x : __int_as_float(0x7fffffff);
}

// The least e in [kMinExp, kMaxExp] with a * 2^up <= 448 * 2^e, a >= 0 finite.  448 = 1.75 * 2^8.
__device__ __forceinline__ int needed_exp(float a, int up) {
  const unsigned bits = __float_as_uint(a);
  const int e =
      static_cast<int>(bits >> 23) - 127 - 8 + up + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(kMinExp, min(kMaxExp, e));
}

// The exponent of the least power of two that is not below a stored scale.
__device__ __forceinline__ int stored_exp(float s) {
  const int bits = __float_as_int(s);
  if (bits <= 0) return kMinExp;
  const int e = (bits >> 23) - 127 + ((bits & 0x7fffff) != 0 ? 1 : 0);
  return max(kMinExp, min(kMaxExp, e));
}

__device__ __forceinline__ uint2 to_e4m3x8(const float (&y)[8], float mul) {
  uint2 r;
  unsigned short h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i] * mul, y[2 * i + 1] * mul),
                                    __NV_SATFINITE, __NV_E4M3);
  }
  r.x = h[0] | (static_cast<uint32_t>(h[1]) << 16);
  r.y = h[2] | (static_cast<uint32_t>(h[3]) << 16);
  return r;
}

__device__ __forceinline__ uint32_t rescale_e4m3x4(uint32_t u, float mul) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw raw =
        __nv_cvt_fp8x2_to_halfraw2(static_cast<unsigned short>(u >> (16 * i)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw));
    r |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(f.x * mul, f.y * mul),
                                                        __NV_SATFINITE, __NV_E4M3))
         << (16 * i);
  }
  return r;
}

// A lane's share of a head row: 16 elements, as two runs of 8 starting at `lo` and `hi`.  Runs are
// laid out so that the two elements of a rotated pair belong to one lane.
struct Unit {
  int lo, hi;
  int angle;  // first column of cos / sin, or -1: these elements are not rotated
};

__device__ __forceinline__ Unit unit_of(int u, int rot, bool interleaved) {
  Unit r;
  if (interleaved || 16 * u >= rot) {
    r.lo = 16 * u;
    r.hi = r.lo + 8;
    r.angle = 16 * u < rot ? 8 * u : -1;
  } else {
    r.lo = 8 * u;
    r.hi = rot / 2 + 8 * u;
    r.angle = 8 * u;
  }
  return r;
}

// Eight angles in packed pairs.
struct Angles {
  uint64_t c[4], s[4];
};

__device__ __forceinline__ void load_angles(Angles& a, const AppendArgs& p, int pos, int col,
                                            float mul) {
  const long long at = static_cast<long long>(pos) * (p.rot_dim / 2) + col;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 c = __ldg(reinterpret_cast<const float4*>(p.cos + at) + i);
    const float4 s = __ldg(reinterpret_cast<const float4*>(p.sin + at) + i);
    a.c[2 * i] = f2_pack(c.x * mul, c.y * mul), a.c[2 * i + 1] = f2_pack(c.z * mul, c.w * mul);
    a.s[2 * i] = f2_pack(s.x * mul, s.y * mul), a.s[2 * i + 1] = f2_pack(s.z * mul, s.w * mul);
  }
}

// The pairs of a lane's 16 elements: first[j], second[j] are the two elements that angle j turns.
__device__ __forceinline__ void split_pairs(const float (&x)[8], const float (&y)[8], bool interleaved,
                                            uint64_t (&first)[4], uint64_t (&second)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (interleaved) {  // neighbours inside each run of 8
      const float(&z)[8] = j < 2 ? x : y;
      first[j] = f2_pack(z[4 * (j & 1)], z[4 * (j & 1) + 2]);
      second[j] = f2_pack(z[4 * (j & 1) + 1], z[4 * (j & 1) + 3]);
    } else {
      first[j] = f2_pack(x[2 * j], x[2 * j + 1]);
      second[j] = f2_pack(y[2 * j], y[2 * j + 1]);
    }
  }
}
__device__ __forceinline__ void join_pairs(float (&x)[8], float (&y)[8], bool interleaved,
                                           const float (&first)[8], const float (&second)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (interleaved) {
      float(&z)[8] = j < 4 ? x : y;
      z[2 * (j & 3)] = first[j];
      z[2 * (j & 3) + 1] = second[j];
    } else {
      x[j] = first[j];
      y[j] = second[j];
    }
  }
}

// Turns a lane's elements, each rounded to odd.
__device__ __forceinline__ void rotate_unit(float (&x)[8], float (&y)[8], const Angles& an,
                                            bool interleaved) {
  uint64_t a[4], b[4];
  float fa[8], fb[8];
  split_pairs(x, y, interleaved, a, b);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t minus_s = f2_mul(an.s[j], kMinusOne2);
    const Sum2 u = sum2(a[j], an.c[j], b[j], minus_s), v = sum2(b[j], an.c[j], a[j], an.s[j]);
    const uint64_t up = f2_fma(a[j], an.c[j], f2_mul(b[j], minus_s));
    const uint64_t vp = f2_fma(b[j], an.c[j], f2_mul(a[j], an.s[j]));
    fa[2 * j] = to_odd(f2_lo(u.hi), f2_lo(u.lo), f2_lo(up));
    fa[2 * j + 1] = to_odd(f2_hi(u.hi), f2_hi(u.lo), f2_hi(up));
    fb[2 * j] = to_odd(f2_lo(v.hi), f2_lo(v.lo), f2_lo(vp));
    fb[2 * j + 1] = to_odd(f2_hi(v.hi), f2_hi(v.lo), f2_hi(vp));
  }
  join_pairs(x, y, interleaved, fa, fb);
}

// Turns a lane's elements to the nearest floats; false where one may not round on to T's nearest: it
// lies halfway between two values of T, is subnormal there, or is not finite.
template <typename T>
__device__ __forceinline__ bool rotate_unit_fast(float (&x)[8], float (&y)[8], const Angles& an,
                                                 bool interleaved) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr uint32_t kBits = kHalf ? 0x1fffu : 0xffffu;  // those that the rounding takes off
  constexpr uint32_t kTie = kHalf ? 0x1000u : 0x8000u;
  uint64_t a[4], b[4], poison = 0;
  float fa[8], fb[8];
  uint32_t tie = 0xffffffffu, small = 0xffffffffu;
  split_pairs(x, y, interleaved, a, b);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t minus_s = f2_mul(an.s[j], kMinusOne2);
    const uint64_t u = sum2(a[j], an.c[j], b[j], minus_s).hi;
    const uint64_t v = sum2(b[j], an.c[j], a[j], an.s[j]).hi;
    poison = f2_fma(u, 0ull, poison);  // 0 times what is not finite
    poison = f2_fma(v, 0ull, poison);
    const uint32_t w[4] = {static_cast<uint32_t>(u), static_cast<uint32_t>(u >> 32),
                           static_cast<uint32_t>(v), static_cast<uint32_t>(v >> 32)};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      tie = min(tie, (w[k] & kBits) ^ kTie);
      if (kHalf) small = min(small, w[k] & 0x7fffffffu);
    }
    fa[2 * j] = f2_lo(u), fa[2 * j + 1] = f2_hi(u);
    fb[2 * j] = f2_lo(v), fb[2 * j + 1] = f2_hi(v);
  }
  const bool sure = tie != 0 && f2_lo(poison) == 0.f && f2_hi(poison) == 0.f &&
                    (!kHalf || small >= 0x38800000u);  // 2^-14
  if (sure) join_pairs(x, y, interleaved, fa, fb);
  return sure;
}

// A lane's 16 elements as they lie in memory.
struct Raw {
  uint4 a, b;
};
template <typename T>
__device__ __forceinline__ Raw load_unit(const T* row, const Unit& u) {
  return Raw{*reinterpret_cast<const uint4*>(row + u.lo), *reinterpret_cast<const uint4*>(row + u.hi)};
}
template <typename T>
__device__ __forceinline__ void widen(const Raw& r, float (&x)[8], float (&y)[8]) {
  const uint32_t wa[4] = {r.a.x, r.a.y, r.a.z, r.a.w}, wb[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 fa = to_float2<T>(wa[i]), fb = to_float2<T>(wb[i]);
    x[2 * i] = fa.x, x[2 * i + 1] = fa.y;
    y[2 * i] = fb.x, y[2 * i + 1] = fb.y;
  }
}

// The sequence of packed row t (t below live_rows): the last s with cu_seqlens[s] <= t.  Each round
// the warp probes 32 places of the range that is left.
__device__ __forceinline__ int find_seq(const int* starts, int n, int t, int lane) {
  int lo = 0;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool below = at < n && starts[lo + at] <= t;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
    lo += last * step;
    n = min(step, n - last * step);
  }
  return lo;
}

// First item of sequence s when each has room for the pages that it can touch: n new tokens touch
// at most n / page + 2 of them, and floor(a + b) - floor(a) >= floor(b).
__device__ __forceinline__ int item_base(const CacheView& c, int s) {
  return (c.cu_seqlens[s] >> c.page_shift) + 2 * s;
}

// The sequence of page item i: the last s with item_base(s) <= i.
__device__ __forceinline__ int find_item_seq(const CacheView& c, int i, int lane) {
  int lo = 0, n = c.n_seqs;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool below = at < n && item_base(c, lo + at) <= i;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
    lo += last * step;
    n = min(step, n - last * step);
  }
  return lo;
}

struct Grid {
  int items;         // page items of one (head, k or v)
  int seq_items;     // of one sequence when all have the same number of new tokens
  int kv_blocks;     // blocks that fill pages; the rest rotate q
  int q_heads;       // heads of q that one lane group takes
  int q_groups;      // lane groups for one token
};

// One page item: the new rows of one page, kv head, and k or v, by WARPS warps together.
template <typename T, int D, int WARPS>
__device__ void fill_page(const AppendArgs& p, const Grid& g, int item, int job, bool active,
                          int tid, float* red) {
  constexpr int kLanes = D / 16;             // lanes for a row
  constexpr int kRows = WARPS * 32 / kLanes;  // rows of one sweep
  constexpr int kKeep = 2;                   // sweeps whose rows stay in registers
  const CacheView& c = p.c;
  const int lane = tid & 31;
  const int head = job >> 1;
  const bool is_v = job & 1;
  const int page_size = 1 << c.page_shift;

  int s, first;  // sequence, first item of the sequence
  if (c.cu_seqlens == nullptr) {
    s = item / g.seq_items;
    first = s * g.seq_items;
  } else {
    s = find_item_seq(c, item, lane);
    first = item_base(c, s);
  }
  const SeqInfo q = seq_info(c, s);
  int begin = q.len - q.n;  // position of the first new token
  int t0 = q.t0;
  if (begin < 0) {  // tokens in front of the cache are not stored
    if (q.n > 0) report_cache_index(c);
    t0 -= begin;
    begin = 0;
  }
  const long long index = (begin >> c.page_shift) + static_cast<long long>(item) - first;
  const long long page_pos = index << c.page_shift;  // position of the page's first slot
  const int a = page_pos < begin ? begin - static_cast<int>(page_pos) : 0;  // first new slot
  const long long left = q.len - page_pos;
  int b = left < page_size ? static_cast<int>(left) : page_size;  // behind the last new slot
  active = active && item >= first && q.n > 0 && b > a;
  const int page = active ? page_of(c, s, static_cast<int>(index)) : -1;
  active = active && page >= 0;
  if (!active) b = a;
  const int rot = !is_v && p.cos != nullptr ? p.rot_dim : 0;
  if (p.cos != nullptr && active && page_pos + b > p.table_rows) {
    report_cache_index(c);  // positions that the table does not have are not stored
    const long long rows = p.table_rows - page_pos;
    b = rows > a ? static_cast<int>(rows) : a;
    active = b > a;
  }

  const int row = tid / kLanes;
  const Unit u = unit_of(tid % kLanes, rot, p.interleaved);
  const T* src = static_cast<const T*>(is_v ? p.v : p.k);
  const long long* st = is_v ? p.sv : p.sk;
  const T* base = src + (t0 + page_pos - begin) * st[0] + head * st[1];  // of slot 0

  // Two bf16 values near the type's largest can rotate past the range of 32 bits: rotated rows are
  // held at half their size.
  const int up = rot > 0 ? 1 : 0;
  const float half = rot > 0 ? 0.5f : 1.f;
  float x[kKeep][8], y[kKeep][8];
  float amax = 0.f;
  auto fetch = [&](int slot, float(&fx)[8], float(&fy)[8]) {
    widen<T>(load_unit<T>(base + slot * st[0], u), fx, fy);
    if (u.angle >= 0) {
      Angles an;
      load_angles(an, p, static_cast<int>(page_pos) + slot, u.angle, half);
      rotate_unit(fx, fy, an, p.interleaved);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        fx[i] *= half;
        fy[i] *= half;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      fx[i] = finite_or_nan(fx[i]);
      fy[i] = finite_or_nan(fy[i]);
      amax = fmaxf(amax, fmaxf(fabsf(fx[i]), fabsf(fy[i])));  // fmaxf passes over NaN
    }
  };
#pragma unroll
  for (int w = 0; w < kKeep; ++w) {
    const int slot = a + row + w * kRows;
    if (slot < b) fetch(slot, x[w], y[w]);
  }
  for (int slot = a + row + kKeep * kRows; slot < b; slot += kRows) {
    float fx[8], fy[8];
    fetch(slot, fx, fy);
  }
  float* scale = (is_v ? c.v_scale : c.k_scale) + (active ? page : 0) * static_cast<long long>(c.Hkv) + head;
  const float old = active && a > 0 ? *scale : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if constexpr (WARPS > 1) {
    if (lane == 0) red[tid >> 5] = amax;
    __syncthreads();  // every job of the block comes here
    amax = red[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) amax = fmaxf(amax, red[i]);
  }
  if (!active) return;
  int e = needed_exp(amax, up);
  if (a > 0) e = max(e, stored_exp(old));
  const float now = pow2f(e);
  const float mul = pow2f(up - e);
  unsigned char* dst = (is_v ? c.v : c.k) + page * (is_v ? c.vs[0] : c.ks[0]) +
                       head * (is_v ? c.vs[1] : c.ks[1]);
  const long long dt = is_v ? c.vs[2] : c.ks[2];
  if (tid == 0) *scale = now;
  if (a > 0 && old != now) {  // earlier rows follow the page's scale
    const float ratio = old * pow2f(-e);
    const int col = (tid % kLanes) * 16;
    for (int slot = row; slot < a; slot += kRows) {
      uint4* at = reinterpret_cast<uint4*>(dst + slot * dt + col);
      uint4 v = *at;
      v.x = rescale_e4m3x4(v.x, ratio);
      v.y = rescale_e4m3x4(v.y, ratio);
      v.z = rescale_e4m3x4(v.z, ratio);
      v.w = rescale_e4m3x4(v.w, ratio);
      *at = v;
    }
  }
  auto put = [&](int slot, const float(&fx)[8], const float(&fy)[8]) {
    unsigned char* at = dst + slot * dt;
    *reinterpret_cast<uint2*>(at + u.lo) = to_e4m3x8(fx, mul);
    *reinterpret_cast<uint2*>(at + u.hi) = to_e4m3x8(fy, mul);
  };
#pragma unroll
  for (int w = 0; w < kKeep; ++w) {
    const int slot = a + row + w * kRows;
    if (slot < b) put(slot, x[w], y[w]);
  }
  for (int slot = a + row + kKeep * kRows; slot < b; slot += kRows) {
    float fx[8], fy[8];
    fetch(slot, fx, fy);
    put(slot, fx, fy);
  }
}

// g.q_heads heads of one packed row of q, by D / 16 lanes.
template <typename T, int D>
__device__ void rotate_q(const AppendArgs& p, const Grid& g, long long group, int lane) {
  constexpr int kLanes = D / 16;
  const CacheView& c = p.c;
  const long long t_ll = group / g.q_groups;
  const int t = t_ll < c.T ? static_cast<int>(t_ll) : c.T;
  const int h0 = static_cast<int>(group - t_ll * g.q_groups) * g.q_heads;
  const int live = live_rows(c);
  int pos = -1;
  // The lanes of a warp hold up to 32 / kLanes rows: find the first one's sequence, then step on.
  const int t_first = __shfl_sync(0xffffffffu, t, 0);
  int s = 0;
  if (c.cu_seqlens == nullptr) {
    s = t / max(1, c.T / c.n_seqs);
  } else if (t_first < live) {
    s = find_seq(c.cu_seqlens, c.n_seqs, t_first, lane);
    while (t < live && s + 1 < c.n_seqs && c.cu_seqlens[s + 1] <= t) ++s;
  }
  if (t >= c.T) return;
  if (t < live && s < c.n_seqs) {
    const SeqInfo q = seq_info(c, s);
    pos = t >= q.t0 && t < q.t0 + q.n ? q.len - q.n + t - q.t0 : -1;
    if (pos < 0 || pos >= p.table_rows) {
      report_cache_index(c);
      pos = -1;
    }
  }
  const Unit u = unit_of(lane % kLanes, p.rot_dim, p.interleaved);
  Angles an;
  if (pos >= 0 && u.angle >= 0) load_angles(an, p, pos, u.angle, 1.f);
  const T* src = static_cast<const T*>(p.q) + t * p.sq[0];
  T* dst = static_cast<T*>(p.q_out) + static_cast<long long>(t) * p.H * D;
  const int h1 = min(p.H, h0 + g.q_heads);
  Raw next = {};
  if (pos >= 0) next = load_unit<T>(src + h0 * p.sq[1], u);
#pragma unroll 1
  for (int h = h0; h < h1; ++h) {
    float x[8], y[8];
    const Raw raw = next;  // zeros without a position
    if (pos >= 0 && h + 1 < h1) next = load_unit<T>(src + (h + 1) * p.sq[1], u);
    widen<T>(raw, x, y);
    if (pos >= 0 && u.angle >= 0 && !rotate_unit_fast<T>(x, y, an, p.interleaved)) {
      rotate_unit(x, y, an, p.interleaved);
    }
    uint4 a, b;
    a.x = from_float2<T>(x[0], x[1]), a.y = from_float2<T>(x[2], x[3]);
    a.z = from_float2<T>(x[4], x[5]), a.w = from_float2<T>(x[6], x[7]);
    b.x = from_float2<T>(y[0], y[1]), b.y = from_float2<T>(y[2], y[3]);
    b.z = from_float2<T>(y[4], y[5]), b.w = from_float2<T>(y[6], y[7]);
    *reinterpret_cast<uint4*>(dst + h * D + u.lo) = a;
    *reinterpret_cast<uint4*>(dst + h * D + u.hi) = b;
  }
}

// Blocks [0, kv_blocks) fill pages, the others rotate q.  ITEM_WARPS warps share a job: a page item
// of one head, k or v.
template <typename T, int D, int THREADS, int ITEM_WARPS>
__global__ void __launch_bounds__(THREADS, 3) fa_cache_append_kernel(
    const __grid_constant__ AppendArgs p, const __grid_constant__ Grid g) {
  constexpr int kPerBlock = THREADS / 32 / ITEM_WARPS;
  __shared__ float red[THREADS / 32];
  const int tid = threadIdx.x;
  if (blockIdx.x < static_cast<unsigned>(g.kv_blocks)) {
    const int sub = tid / (32 * ITEM_WARPS);
    const long long id = static_cast<long long>(blockIdx.x) * kPerBlock + sub;
    const int jobs = 2 * p.c.Hkv;
    const long long item = id / jobs;
    const bool active = item < g.items;
    fill_page<T, D, ITEM_WARPS>(p, g, active ? static_cast<int>(item) : 0,
                                static_cast<int>(id - item * jobs), active,
                                tid % (32 * ITEM_WARPS), red + sub * ITEM_WARPS);
  } else {
    const long long group =
        (static_cast<long long>(blockIdx.x - g.kv_blocks) * THREADS + tid) / (D / 16);
    rotate_q<T, D>(p, g, group, tid & 31);
  }
}

template <typename T, int D>
cudaError_t launch_t(const AppendArgs& a, cudaStream_t stream) {
  constexpr int kLanes = D / 16;
  const CacheView& c = a.c;
  const int page = 1 << c.page_shift;
  Grid g;
  const int mean = c.T / c.n_seqs;
  long long items;
  if (c.cu_seqlens == nullptr) {
    g.seq_items = mean <= 1 ? 1 : (mean - 2) / page + 2;
    items = static_cast<long long>(g.seq_items) * c.n_seqs;
  } else {
    g.seq_items = 0;
    items = c.T / page + 2ll * c.n_seqs;
  }
  if (items > 0x7fffffffll) return cudaErrorInvalidValue;
  g.items = static_cast<int>(items);
  // Few rows of a page come at a time: a warp for each job.  Else as many warps as hold a page's rows
  // of one head in registers, 32 values a thread: with more, most of a block's time is its chain of
  // lookups (eight warps for any page: 102 us for 16384 tokens of 12 heads of 64, pages of 32).
  const int warps = mean < 8 ? 1 : std::min(8, page * D / 1024);
  const int threads = 256;
  const int per_block = threads / 32 / warps;
  const long long kv_blocks = (items * 2 * c.Hkv + per_block - 1) / per_block;
  long long q_blocks = 0;
  g.q_heads = 1;
  g.q_groups = 1;
  if (a.q != nullptr) {
    const long long rows = static_cast<long long>(c.T) * a.H;
    const long long fill = static_cast<long long>(multiprocessors()) * 1024 / kLanes;
    while (g.q_heads < 8 && g.q_heads < a.H && rows / (2 * g.q_heads) >= fill) g.q_heads *= 2;
    g.q_groups = (a.H + g.q_heads - 1) / g.q_heads;
    q_blocks = (static_cast<long long>(c.T) * g.q_groups * kLanes + threads - 1) / threads;
  }
  if (kv_blocks + q_blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  g.kv_blocks = static_cast<int>(kv_blocks);
  const unsigned blocks = static_cast<unsigned>(kv_blocks + q_blocks);
  switch (warps) {
    case 1: fa_cache_append_kernel<T, D, 256, 1><<<blocks, 256, 0, stream>>>(a, g); break;
    case 2: fa_cache_append_kernel<T, D, 256, 2><<<blocks, 256, 0, stream>>>(a, g); break;
    case 4: fa_cache_append_kernel<T, D, 256, 4><<<blocks, 256, 0, stream>>>(a, g); break;
    default: fa_cache_append_kernel<T, D, 256, 8><<<blocks, 256, 0, stream>>>(a, g); break;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_cache_append(const AppendArgs& a, cudaStream_t stream) {
  if (a.dtype == FA_DTYPE_F16) {
    return a.D == 64 ? launch_t<__half, 64>(a, stream) : launch_t<__half, 128>(a, stream);
  }
  return a.D == 64 ? launch_t<__nv_bfloat16, 64>(a, stream)
                   : launch_t<__nv_bfloat16, 128>(a, stream);
}

}  // namespace fa_sm100
