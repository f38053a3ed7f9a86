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
// What is stored or returned is the rounding of the exact rotated value, whatever the order of
// operations: a c + b s is computed in 32 bits with a bound w on its error, and where a c + b s - w and
// a c + b s + w round to the same 8 or 16 bits, that is it.  Where they do not (a value next to a border:
// one of some 2^12 for bf16, 2^9 for fp16, 2^18 for e4m3) the sum is done over as an unevaluated
// sum of two floats, both products exactly (their errors by fma), the sum's error by the two-sum of
// Knuth, rounded to odd in 32 bits (the last bit set where it is inexact), so that the rounding that
// follows is that of the exact value.  (Products below 2^-102, whose own error leaves a float's range, aside.)
// A page's scale is settled likewise, by bounds on its largest magnitude.  13613 tokens of 32 + 8 + 8 heads of 128, where the memory needs 47 us: 64-bit arithmetic
// 129 us (conversions, 16 a cycle), every sum as two floats or these bounds 105 to 113 us (q alone 54, k
// and v 59, of which the rotation 36: instructions bound it, not the memory).
#include <algorithm>
#include <cmath>

#include "fa_cache_common.cuh"
#include "sm100_ptx.cuh"

namespace fa_sm100 {
namespace {

constexpr int kThreads = 256;
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

// a b rounded to odd.
__device__ __forceinline__ float times_odd(float a, float b) {
  const float p = a * b;
  return to_odd(p, fmaf(a, b, -p), p);
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

// Two values; what is not finite has to be NaN before (infinities saturate).
__device__ __forceinline__ uint32_t to_e4m3x2(uint64_t v) {
  return __nv_cvt_float2_to_fp8x2(make_float2(f2_lo(v), f2_hi(v)), __NV_SATFINITE, __NV_E4M3);
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

// `mul` has 24 bits where the scale was no power of two, and then a float does not hold its products.
__device__ __forceinline__ uint32_t rescale_e4m3x4(uint32_t u, float mul) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw raw =
        __nv_cvt_fp8x2_to_halfraw2(static_cast<unsigned short>(u >> (16 * i)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw));
    r |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(times_odd(f.x, mul), times_odd(f.y, mul)),
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

// Eight angles in packed pairs, and 3.125 * 2^-24 of the largest |cos| or |sin| among them.
struct Angles {
  uint64_t c[4], s[4], minus_s[4];
  float eps;
};

__device__ __forceinline__ void load_angles(Angles& a, const AppendArgs& p, int pos, int col,
                                            float mul) {
  const long long at = static_cast<long long>(pos) * (p.rot_dim / 2) + col;
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 c = __ldg(reinterpret_cast<const float4*>(p.cos + at) + i);
    const float4 s = __ldg(reinterpret_cast<const float4*>(p.sin + at) + i);
    a.c[2 * i] = f2_pack(c.x * mul, c.y * mul), a.c[2 * i + 1] = f2_pack(c.z * mul, c.w * mul);
    a.s[2 * i] = f2_pack(s.x * mul, s.y * mul), a.s[2 * i + 1] = f2_pack(s.z * mul, s.w * mul);
    big = fmax3(big, fmax3(fabsf(c.x), fabsf(c.y), fmaxf(fabsf(c.z), fabsf(c.w))),
                fmax3(fabsf(s.x), fabsf(s.y), fmaxf(fabsf(s.z), fabsf(s.w))));
  }
  a.eps = big * mul * 0x1.9p-23f;
#pragma unroll
  for (int j = 0; j < 4; ++j) a.minus_s[j] = f2_mul(a.s[j], kMinusOne2);
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
__device__ __forceinline__ uint64_t f2_abs(uint64_t x) { return x & 0x7fffffff7fffffffull; }

// Pair j turned in plain 32 bits, and a bound on how far the values and the values +- w are off: a
// product, the fma and the sum with w round once each, 2^-24 (|b s| + 2 |a c + b s|) in all, which is at
// most 3 * 2^-24 (|a| + |b|) times the largest |c| or |s|.
struct Bounded {
  uint64_t x, y, w;
};
__device__ __forceinline__ Bounded turn_bounded(uint64_t a, uint64_t b, const Angles& an, int j) {
  return Bounded{f2_fma(a, an.c[j], f2_mul(b, an.minus_s[j])), f2_fma(b, an.c[j], f2_mul(a, an.s[j])),
                 f2_mul(f2_add(f2_abs(a), f2_abs(b)), f2_pack(an.eps, an.eps))};
}

// The same rounded to odd.
__device__ __forceinline__ void turn_odd(uint64_t a, uint64_t b, const Angles& an, int j, float (&fa)[2],
                                         float (&fb)[2]) {
  const Sum2 u = sum2(a, an.c[j], b, an.minus_s[j]), v = sum2(b, an.c[j], a, an.s[j]);
  const Bounded p = turn_bounded(a, b, an, j);
  fa[0] = to_odd(f2_lo(u.hi), f2_lo(u.lo), f2_lo(p.x));
  fa[1] = to_odd(f2_hi(u.hi), f2_hi(u.lo), f2_hi(p.x));
  fb[0] = to_odd(f2_lo(v.hi), f2_lo(v.lo), f2_lo(p.y));
  fb[1] = to_odd(f2_hi(v.hi), f2_hi(v.lo), f2_hi(p.y));
}

template <typename T>
__device__ __forceinline__ uint32_t narrow2(uint64_t v) {
  return from_float2<T>(f2_lo(v), f2_hi(v));
}

// Turns a lane's elements and rounds them to T: the words of its two runs.
template <typename T>
__device__ __forceinline__ void rotate_to(const float (&x)[8], const float (&y)[8], const Angles& an,
                                          bool interleaved, uint32_t (&wx)[4], uint32_t (&wy)[4]) {
  uint64_t a[4], b[4];
  split_pairs(x, y, interleaved, a, b);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const Bounded t = turn_bounded(a[j], b[j], an, j);
    uint32_t fu = narrow2<T>(f2_add(t.x, t.w)), fv = narrow2<T>(f2_add(t.y, t.w));
    const uint32_t gu = narrow2<T>(f2_fma(t.w, kMinusOne2, t.x));
    const uint32_t gv = narrow2<T>(f2_fma(t.w, kMinusOne2, t.y));
    if (((fu ^ gu) | (fv ^ gv)) != 0) {
      float p[2], q[2];
      turn_odd(a[j], b[j], an, j, p, q);
      fu = from_float2<T>(p[0], p[1]);
      fv = from_float2<T>(q[0], q[1]);
    }
    if (interleaved) {
      uint32_t(&w)[4] = j < 2 ? wx : wy;
      w[2 * (j & 1)] = __byte_perm(fu, fv, 0x5410);
      w[2 * (j & 1) + 1] = __byte_perm(fu, fv, 0x7632);
    } else {
      wx[j] = fu;
      wy[j] = fv;
    }
  }
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

// The sequence of packed row t, if it is one's: the last s with cu_seqlens[s] <= t.  Each round the warp
// probes 32 places of the range that is left.  Compared without signs, so that a negative offset is not
// below: an offset out of range then costs the sequences that it bounds and, among up to 32, no other.
__device__ __forceinline__ int find_seq(const int* starts, int n, int t, int lane) {
  int lo = 0;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool below = at < n && static_cast<unsigned>(starts[lo + at]) <= static_cast<unsigned>(t);
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

// The sequence of page item i: the last s with item_base(s) <= i, of those that begin in the batch (find_seq).
__device__ __forceinline__ int find_item_seq(const CacheView& c, int i, int lane) {
  int lo = 0, n = c.n_seqs;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool below = at < n && static_cast<unsigned>(c.cu_seqlens[lo + at]) <= static_cast<unsigned>(c.T) &&
                       item_base(c, lo + at) <= i;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
    lo += last * step;
    n = min(step, n - last * step);
  }
  return lo;
}

struct Grid {
  int items;         // page items of one (head, k or v)
  int seq_items;     // of one sequence when all have the same number of new tokens
  int kv_blocks;     // blocks that fill pages; in one launch the rest rotate q
  int q_heads;       // heads of q that one lane group takes
  int q_groups;      // lane groups for one token
};

// One page item: the new rows of one page, kv head, and k or v, by WARPS warps together.
template <typename T, int D, int WARPS, bool ROTATES>
__device__ __forceinline__ void fill_page(const AppendArgs& p, const Grid& g, int item, int job, bool active,
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
  // Of a length past the table's room the tokens that have a page are stored where they belong.
  const SeqInfo q = seq_info<true>(c, s);
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
  const int rot = ROTATES && !is_v ? p.rot_dim : 0;
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
  // taken at half their size.
  const int up = rot > 0 ? 1 : 0;
  const float half = rot > 0 ? 0.5f : 1.f;
  const bool turns = ROTATES && u.angle >= 0;
  Raw kept[kKeep] = {};
  float amax = 0.f, off = 0.f;  // the largest magnitude, and a bound on its error
  auto look = [&](int slot, const Raw& raw) {
    float x[8], y[8];
    widen<T>(raw, x, y);
    if (turns) {
      Angles an;
      load_angles(an, p, static_cast<int>(page_pos) + slot, u.angle, half);
      uint64_t pa[4], pb[4];
      split_pairs(x, y, p.interleaved, pa, pb);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Bounded t = turn_bounded(pa[j], pb[j], an, j);
        amax = fmax3(amax, fabsf(f2_lo(t.x)), fabsf(f2_hi(t.x)));  // passes over NaN
        amax = fmax3(amax, fabsf(f2_lo(t.y)), fabsf(f2_hi(t.y)));
        off = fmax3(off, f2_lo(t.w), f2_hi(t.w));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float fx = fabsf(finite_or_nan(x[i] * half)), fy = fabsf(finite_or_nan(y[i] * half));
        amax = fmax3(amax, fx, fy);
      }
    }
  };
  // The same exactly, where the bounds leave the scale open or a value is not finite.
  auto look_again = [&](int slot, const Raw& raw) {
    float x[8], y[8];
    widen<T>(raw, x, y);
    if (turns) {
      Angles an;
      load_angles(an, p, static_cast<int>(page_pos) + slot, u.angle, half);
      uint64_t pa[4], pb[4];
      split_pairs(x, y, p.interleaved, pa, pb);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float fa[2], fb[2];
        turn_odd(pa[j], pb[j], an, j, fa, fb);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          amax = fmax3(amax, fabsf(finite_or_nan(fa[k])), fabsf(finite_or_nan(fb[k])));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float fx = fabsf(finite_or_nan(x[i] * half)), fy = fabsf(finite_or_nan(y[i] * half));
        amax = fmax3(amax, fx, fy);
      }
    }
  };
#pragma unroll
  for (int w = 0; w < kKeep; ++w) {
    const int slot = a + row + w * kRows;
    if (slot < b) kept[w] = load_unit<T>(base + slot * st[0], u);
  }
#pragma unroll
  for (int w = 0; w < kKeep; ++w) {
    const int slot = a + row + w * kRows;
    if (slot < b) look(slot, kept[w]);
  }
#pragma unroll 1
  for (int slot = a + row + kKeep * kRows; slot < b; slot += kRows) {
    look(slot, load_unit<T>(base + slot * st[0], u));
  }
  float* scale = (is_v ? c.v_scale : c.k_scale) + (active ? page : 0) * static_cast<long long>(c.Hkv) + head;
  const float old = active && a > 0 ? *scale : 0.f;
  auto group_max = [&](float v) {  // over the job's warps; the block comes here together
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (WARPS > 1) {
      __syncthreads();  // the last values were read
      if (lane == 0) red[tid >> 5] = v;
      __syncthreads();
      v = red[0];
#pragma unroll
      for (int i = 1; i < WARPS; ++i) v = fmaxf(v, red[i]);
    }
    return v;
  };
  amax = group_max(amax);
  if (ROTATES) {
    off = group_max(off);
    // amax + off may be infinite, which no exponent equals.
    const bool open = needed_exp(amax + off, up) != needed_exp(fmaxf(amax - off, 0.f), up) ||
                      !(amax + off < INFINITY);
    if (WARPS > 1 ? __syncthreads_or(open) : __any_sync(0xffffffffu, open)) {
      if (open) amax = 0.f;
#pragma unroll 1
      for (int slot = a + row; slot < b && open; slot += kRows) {
        look_again(slot, load_unit<T>(base + slot * st[0], u));
      }
      amax = group_max(amax);
    }
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
  auto put = [&](int slot, const Raw& raw) {
    unsigned char* at = dst + slot * dt;
    float x[8], y[8];
    widen<T>(raw, x, y);
    uint2 wx, wy;
    if (turns) {
      Angles an;
      load_angles(an, p, static_cast<int>(page_pos) + slot, u.angle, half);
      uint64_t pa[4], pb[4];
      split_pairs(x, y, p.interleaved, pa, pb);
      const uint64_t mul2 = f2_pack(mul, mul);
      uint32_t h[8];  // pairs of bytes: run lo, then run hi
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Bounded t = turn_bounded(pa[j], pb[j], an, j);
        uint32_t f = to_e4m3x2(f2_mul(f2_add(t.x, t.w), mul2));
        uint32_t g2 = to_e4m3x2(f2_mul(f2_add(t.y, t.w), mul2));
        const uint32_t f1 = to_e4m3x2(f2_mul(f2_fma(t.w, kMinusOne2, t.x), mul2));
        const uint32_t g1 = to_e4m3x2(f2_mul(f2_fma(t.w, kMinusOne2, t.y), mul2));
        if (((f ^ f1) | (g2 ^ g1)) != 0) {
          float fa[2], fb[2];
          turn_odd(pa[j], pb[j], an, j, fa, fb);
          f = to_e4m3x2(f2_pack(finite_or_nan(fa[0]) * mul, finite_or_nan(fa[1]) * mul));
          g2 = to_e4m3x2(f2_pack(finite_or_nan(fb[0]) * mul, finite_or_nan(fb[1]) * mul));
        }
        if (p.interleaved) {
          h[2 * j] = __byte_perm(f, g2, 0x0040);      // bytes f0, g0
          h[2 * j + 1] = __byte_perm(f, g2, 0x0051);  // f1, g1
        } else {
          h[j] = f;
          h[4 + j] = g2;
        }
      }
      wx = make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
      wy = make_uint2(__byte_perm(h[4], h[5], 0x5410), __byte_perm(h[6], h[7], 0x5410));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = finite_or_nan(x[i] * half);
        y[i] = finite_or_nan(y[i] * half);
      }
      wx = to_e4m3x8(x, mul);
      wy = to_e4m3x8(y, mul);
    }
    *reinterpret_cast<uint2*>(at + u.lo) = wx;
    *reinterpret_cast<uint2*>(at + u.hi) = wy;
  };
#pragma unroll
  for (int w = 0; w < kKeep; ++w) {
    const int slot = a + row + w * kRows;
    if (slot < b) put(slot, kept[w]);
  }
#pragma unroll 1
  for (int slot = a + row + kKeep * kRows; slot < b; slot += kRows) {
    put(slot, load_unit<T>(base + slot * st[0], u));
  }
}

// g.q_heads heads of one packed row of q, by D / 16 lanes.
template <typename T, int D>
__device__ __forceinline__ void rotate_q(const AppendArgs& p, const Grid& g, long long group, int lane) {
  constexpr int kLanes = D / 16;
  const CacheView& c = p.c;
  const long long t_ll = group / g.q_groups;
  const int t = t_ll < c.T ? static_cast<int>(t_ll) : c.T;
  const int h0 = static_cast<int>(group - t_ll * g.q_groups) * g.q_heads;
  const Unit u = unit_of(lane % kLanes, p.rot_dim, p.interleaved);
  const T* src = static_cast<const T*>(p.q) + t * p.sq[0];
  T* dst = static_cast<T*>(p.q_out) + static_cast<long long>(t) * p.H * D;
  const int h1 = t < c.T ? min(p.H, h0 + g.q_heads) : h0;
  // Four heads' rows in flight, the first ones while the row's position is looked up.
  constexpr int kAhead = 4;
  Raw ring[kAhead] = {};
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    if (h0 + i < h1) ring[i] = load_unit<T>(src + (h0 + i) * p.sq[1], u);
  }
  int pos = -1;
  // The lanes of a warp hold up to 32 / kLanes rows: find the first one's sequence, then step on.
  const int t_first = __shfl_sync(0xffffffffu, t, 0);
  int s = 0;
  if (c.cu_seqlens == nullptr) {
    s = t / max(1, c.T / c.n_seqs);
  } else if (t_first < c.T) {
    s = find_seq(c.cu_seqlens, c.n_seqs, t_first, lane);
    for (int next = s + 1; next < c.n_seqs; ++next) {
      const int start = c.cu_seqlens[next];
      if (start > t && start <= c.T) break;
      if (start >= 0 && start <= t) s = next;
    }
  }
  if (t >= c.T) return;
  if (s < c.n_seqs) {
    const SeqInfo q = seq_info<true>(c, s);
    if (t >= q.t0 && t < q.t0 + q.n) {  // else a row of no sequence
      pos = q.len - q.n + (t - q.t0);  // below len, which may be any int
      if (pos < 0 || pos >= p.table_rows) {
        report_cache_index(c);
        pos = -1;
      }
    }
  }
  Angles an;
  if (pos >= 0 && u.angle >= 0) load_angles(an, p, pos, u.angle, 1.f);
#pragma unroll 1
  for (int hb = h0; hb < h1; hb += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = hb + i;
      if (h >= h1) break;
      const Raw raw = ring[i];
      if (h + kAhead < h1) ring[i] = load_unit<T>(src + (h + kAhead) * p.sq[1], u);
      uint32_t wx[4] = {raw.a.x, raw.a.y, raw.a.z, raw.a.w};
      uint32_t wy[4] = {raw.b.x, raw.b.y, raw.b.z, raw.b.w};
      if (pos < 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) wx[k] = wy[k] = 0;
      } else if (u.angle >= 0) {
        float x[8], y[8];
        widen<T>(raw, x, y);
        rotate_to<T>(x, y, an, p.interleaved, wx, wy);
      }
      *reinterpret_cast<uint4*>(dst + h * D + u.lo) = make_uint4(wx[0], wx[1], wx[2], wx[3]);
      *reinterpret_cast<uint4*>(dst + h * D + u.hi) = make_uint4(wy[0], wy[1], wy[2], wy[3]);
    }
  }
}

// ITEM_WARPS warps share a job: a page item of one head, k or v.
template <typename T, int D, int ITEM_WARPS, bool ROTATES>
__device__ __forceinline__ void fill_block(const AppendArgs& p, const Grid& g, int block) {
  constexpr int kPerBlock = kThreads / 32 / ITEM_WARPS;
  __shared__ float red[kThreads / 32];
  const int sub = threadIdx.x / (32 * ITEM_WARPS);
  const long long id = static_cast<long long>(block) * kPerBlock + sub;
  const int jobs = 2 * p.c.Hkv;
  const long long item = id / jobs;
  const bool active = item < g.items;
  fill_page<T, D, ITEM_WARPS, ROTATES>(p, g, active ? static_cast<int>(item) : 0,
                                       static_cast<int>(id - item * jobs), active,
                                       threadIdx.x % (32 * ITEM_WARPS), red + sub * ITEM_WARPS);
  if (block == 0 && p.c.cu_seqlens != nullptr) {  // offsets that are out of order may hide each other from the items
    for (int s = threadIdx.x; s < p.c.n_seqs; s += kThreads) {
      if (!offsets_ok(p.c, s, p.c.cu_seqlens[s], p.c.cu_seqlens[s + 1])) report_cache_index(p.c);
    }
  }
}
template <typename T, int D>
__device__ __forceinline__ void rotate_block(const AppendArgs& p, const Grid& g, int block) {
  rotate_q<T, D>(p, g, (static_cast<long long>(block) * kThreads + threadIdx.x) / (D / 16),
                 threadIdx.x & 31);
}

// One launch, a warp for each job: blocks [0, kv_blocks) fill pages, the others rotate q.
template <typename T, int D, bool ROTATES>
__global__ void __launch_bounds__(kThreads) fa_cache_append_kernel(
    const __grid_constant__ AppendArgs p, const __grid_constant__ Grid g) {
  const int block = blockIdx.x;
  if (block < g.kv_blocks) {
    fill_block<T, D, 1, ROTATES>(p, g, block);
  } else if (ROTATES) {
    rotate_block<T, D>(p, g, block - g.kv_blocks);
  }
}

// A launch each, several warps for a job.  They need nothing of each other and run together.
template <typename T, int D, int ITEM_WARPS, bool ROTATES>
__global__ void __launch_bounds__(kThreads, 3) fa_cache_fill_kernel(
    const __grid_constant__ AppendArgs p, const __grid_constant__ Grid g) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  fill_block<T, D, ITEM_WARPS, ROTATES>(p, g, blockIdx.x);
}
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) fa_cache_turn_kernel(
    const __grid_constant__ AppendArgs p, const __grid_constant__ Grid g) {
  rotate_block<T, D>(p, g, blockIdx.x);
  wait_for_parts();  // done only when the pages are
}

template <typename T, int D, int WARPS>
void launch_fill(const AppendArgs& a, const Grid& g, unsigned blocks, cudaStream_t stream) {
  if (a.cos != nullptr) {
    fa_cache_fill_kernel<T, D, WARPS, true><<<blocks, kThreads, 0, stream>>>(a, g);
  } else {
    fa_cache_fill_kernel<T, D, WARPS, false><<<blocks, kThreads, 0, stream>>>(a, g);
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
  // A job (a page item of one head, k or v) costs its warps a chain of lookups and then its rows one
  // sweep after the other.  With many jobs for their rows a warp for each, and q in the same launch:
  // the chains of many jobs hide each other, and a block waits for nothing.  With few, as many warps as
  // hold a page's rows in registers, 32 values a thread, and a launch for q.  Measured, us, a warp / more:
  // 16 x 1024 tokens of 12 heads of 64, pages of 32 (12672 jobs) 18 / 24; 64 x 64 of 32 + 8 heads of 128,
  // pages of 64 (2048) 32 / 41; 2048, pages of 32 (1072) 18 / 20, of 64 (544) 26 / 19, of 128 (288) 48 / 20;
  // 64 x 128, pages of 128 (2048) 81 / 69.  A job's time goes with its rows and D, and so does the border.
  const long long jobs = items * 2 * c.Hkv;
  const bool one_launch = mean < 8 || jobs >= static_cast<long long>(std::min(mean, page)) * D / 4;
  const int warps = one_launch ? 1 : std::min(8, page * D / 1024);
  const int per_block = kThreads / 32 / warps;
  const long long kv_blocks = (jobs + per_block - 1) / per_block;
  long long q_blocks = 0;
  g.q_heads = 1;
  g.q_groups = 1;
  if (a.q != nullptr) {
    const long long rows = static_cast<long long>(c.T) * a.H;
    const long long fill = static_cast<long long>(multiprocessors()) * 512 / kLanes;
    while (g.q_heads < a.H && rows / (2 * g.q_heads) >= fill) g.q_heads *= 2;
    g.q_groups = (a.H + g.q_heads - 1) / g.q_heads;
    q_blocks = (static_cast<long long>(c.T) * g.q_groups * kLanes + kThreads - 1) / kThreads;
  }
  if (kv_blocks + q_blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  g.kv_blocks = static_cast<int>(kv_blocks);
  const bool turns = a.cos != nullptr;
  if (one_launch) {
    const unsigned blocks = static_cast<unsigned>(kv_blocks + q_blocks);
    if (turns) {
      fa_cache_append_kernel<T, D, true><<<blocks, kThreads, 0, stream>>>(a, g);
    } else {
      fa_cache_append_kernel<T, D, false><<<blocks, kThreads, 0, stream>>>(a, g);
    }
    return cudaGetLastError();
  }
  const unsigned blocks = static_cast<unsigned>(kv_blocks);
  switch (warps) {
    case 1: launch_fill<T, D, 1>(a, g, blocks, stream); break;
    case 2: launch_fill<T, D, 2>(a, g, blocks, stream); break;
    case 4: launch_fill<T, D, 4>(a, g, blocks, stream); break;
    default: launch_fill<T, D, 8>(a, g, blocks, stream); break;
  }
  if (q_blocks > 0) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(q_blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fa_cache_turn_kernel<T, D>, a, g);
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
