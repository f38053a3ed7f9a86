// fa_cache_attn.cu -- attention of packed new tokens over a paged cache held in e4m3 with a scale
// for each (page, kv head).  No counterpart in the reference, which has no cache; the recurrence and
// the conventions of an empty row (O = 0, LSE = +inf) are the forward's.
//
// Query row i of sequence s sees the keys j < len (full) or j <= len - n + i (causal: the new tokens
// are the sequence's last ones).  With K_j = sk_j kq_j and V_j = sv_j vq_j (kq, vq in e4m3, the
// scales constant over a page), all in units of log2:
//   t_j = scale * log2(e) * sk_j * (q . kq_j) + log2(sv_j),   m = max t_j,   P_j = 2^(t_j - m) <= 1
//   O = sum_j P_j vq_j / l,   l = sum_j P_j / sv_j,   LSE = (m + log2 l) ln 2.
// Folding V's scale into the exponent keeps P in 16 bits' range whatever the scales are, leaves the
// products to plain e4m3 values (exact in fp16, so one fp16 product form serves fp16 and bf16
// queries), and costs one term for a run of 16 keys, since a run never leaves its page.
//
// bf16 queries enter the products as fp16 after division by a power of two for each row: 8
// significant bits fit in fp16's 11, so this is exact but for values 2^-23 below the row's largest.
#include <algorithm>
#include <cmath>

#include "fa_cache_common.cuh"
#include "sm100_ptx.cuh"

namespace fa_sm100 {
namespace {

constexpr int kRows = 16;   // query rows (token, head of the group) of one tile
constexpr int kRun = 16;    // keys that a warp takes at a time; never more than a page
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = kRun * kWarps;  // keys of one unit of work
constexpr int kStages = 4;            // runs in flight for each warp
constexpr int kPerSm = 3;             // CTAs on a multiprocessor
constexpr float kLazy = 8.0f;         // the running maximum follows once it is off by 2^8
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct Layout {
  static constexpr int kHalf = kRun * D;  // K or V bytes of a run
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kMerge = kWarps * kRows * D * 4;  // reuses the ring
  static constexpr int kMain = kRing > kMerge ? kRing : kMerge;
  static constexpr int kScale = kWarps * kStages * 16;
  static constexpr int kBars = kWarps * kStages * 8;
  static constexpr int kBytes = kMain + kScale + kBars + 1024;  // the ring starts on 1024 bytes
};

// A partial result: kRows x D sums, then (m, l) of each row.
__host__ __device__ constexpr int partial_floats(int D) { return kRows * D + 2 * kRows; }

// Work of a sequence: row tiles x kv heads tuples, each of `tiles` units (at least one, so that a
// row without keys is written too).
struct SeqWork {
  SeqInfo q;
  int row_tiles;
  int tiles;
  __device__ long long units(int Hkv) const {
    return static_cast<long long>(row_tiles) * Hkv * tiles;
  }
};

__device__ __forceinline__ SeqWork seq_work(const CacheView& c, int s, int group) {
  SeqWork w;
  w.q = seq_info(c, s);
  w.row_tiles = (w.q.n * group + kRows - 1) / kRows;
  w.tiles = max(1, (w.q.len + kTile - 1) / kTile);
  return w;
}

// Units are numbered sequence by sequence; CTA i takes [bound(i), bound(i + 1)), never none: no more
// CTAs work than there are units.
__device__ __forceinline__ int ctas_of(long long total) {
  return static_cast<int>(min(total, static_cast<long long>(gridDim.x)));
}
__device__ __forceinline__ long long bound_of(long long total, int i, int ctas) {
  return total * i / ctas;
}

struct Place {
  int s;            // sequence of the unit
  long long first;  // its first unit
};

template <int THREADS>
__device__ long long block_sum(long long x, long long* tmp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) x += tmp[i];
  return x;
}

// The total of units, then the sequence that holds one of them.
template <int THREADS>
struct Finder {
  long long warp[THREADS / 32];
  Place at;

  __device__ long long total(const CacheView& c, int group) {
    if (threadIdx.x == 0) at = Place{0, 0};
    long long sum = 0;
    for (int s = threadIdx.x; s < c.n_seqs; s += THREADS) sum += seq_work(c, s, group).units(c.Hkv);
    return block_sum<THREADS>(sum, warp);
  }

  __device__ void find(const CacheView& c, int group, long long target) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    long long run = 0;
    for (int base = 0; base < c.n_seqs; base += THREADS) {
      const int s = base + threadIdx.x;
      const long long mine = s < c.n_seqs ? seq_work(c, s, group).units(c.Hkv) : 0;
      long long incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      __syncthreads();
      if (lane == 31) warp[wid] = incl;
      __syncthreads();
      long long before = run;
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) {
        if (i < wid) before += warp[i];
        run += warp[i];
      }
      incl += before;
      if (mine > 0 && target >= incl - mine && target < incl) at = Place{s, incl - mine};
    }
    __syncthreads();
  }
};

// Bounded wait for a phase of this warp's copies; false when the time limit ran out (reported).
__device__ __forceinline__ bool wait_copy(uint32_t bar, uint32_t parity, const CacheAttnArgs& a) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > a.timeout_ns) {
      atomicOr(a.c.status, kStKFull);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}

// Two e4m3 values (the low or high half of u) as fp16.
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t u) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(u));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t u) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(u));
  return r;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a run's scores need: t = s * mul + add, l += sum * inv.
struct RunScale {
  float mul, add, inv;
  int present;
};

// A page's value scale as (log2, reciprocal); exact for powers of two.  Scales are positive; zero
// and subnormal ones count as 2^-64, which leaves the keys in the denominator and adds nothing.
__device__ __forceinline__ void value_scale(float s, float* add, float* inv) {
  s = s != s ? s : fminf(fmaxf(s, 0x1p-64f), 0x1p120f);
  const int bits = __float_as_int(s);
  const float mant = __int_as_float((bits & 0x7fffff) | 0x3f800000);
  *add = static_cast<float>((bits >> 23) - 127) + log2f(mant);
  *inv = 1.0f / s;
}

// Copies 16 keys of a page and head to shared memory, 128- or 64-byte swizzled (a row's 16-byte piece
// p lies at p ^ (row & 7), or p ^ ((row >> 1) & 3) for rows of 64 bytes).
__device__ __forceinline__ void load_page(uint32_t dst, const void* map, int pos, int slot, int head,
                                          int page, uint32_t bar) {
  const int pt = pos & 3, ph = (pos >> 2) & 3;
  const int c0 = pt == 0 ? slot : (ph == 0 ? head : page);
  const int c1 = pt == 1 ? slot : (ph == 1 ? head : page);
  const int c2 = pt == 2 ? slot : (ph == 2 ? head : page);
  tma_load_4d(dst, map, 0, c0, c1, c2, bar);
}

// The 16-byte pieces of a K row that lane column cq multiplies: neighbours, so that the eight lanes
// of a shared-memory phase (two rows) read all eight pieces.
template <int D>
__device__ __forceinline__ int k_piece(int cq, int p) {
  return (D / 64) * cq + p;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kPerSm) fa_cache_decode_kernel(
    const __grid_constant__ CacheAttnArgs a, const __grid_constant__ PageMaps maps,
    float* partials) {
  using L = Layout<D>;
  constexpr int kSteps = D / 16;       // products of 16 along D
  constexpr int kWords = D / 16;       // 4-byte words of a K row that a lane holds
  constexpr int kPieces = D / 16;      // 16-byte pieces of a row
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ Finder<kThreads> finder;
  __shared__ float merge_m[kWarps][kRows], merge_l[kWarps][kRows];

  const CacheView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = lane >> 2, cq = lane & 3;  // row (and key) group, column group of the fragments
  const int group = a.H / c.Hkv;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // Rows behind the last sequence.
  {
    const int live = live_rows(c);
    const long long n = static_cast<long long>(c.T - live) * a.H;
    T* o = static_cast<T*>(a.o) + static_cast<long long>(live) * a.H * D;
    for (long long i = static_cast<long long>(blockIdx.x) * kThreads + tid; i < n * (D / 8);
         i += static_cast<long long>(gridDim.x) * kThreads) {
      reinterpret_cast<uint4*>(o)[i] = make_uint4(0, 0, 0, 0);
      if (i % (D / 8) == 0) a.lse[static_cast<long long>(live) * a.H + i / (D / 8)] = 0.f;
    }
  }

  const long long total = finder.total(c, group);
  const int ctas = ctas_of(total);
  if (blockIdx.x >= static_cast<unsigned>(ctas)) return;
  const long long u_begin = bound_of(total, blockIdx.x, ctas);
  const long long u_end = bound_of(total, blockIdx.x + 1, ctas);
  finder.find(c, group, u_begin);
  int s = finder.at.s;
  long long seq_first = finder.at.first;

  const uint32_t ring = smem_u32(smem) + warp * kStages * L::kStage;
  RunScale* scales = reinterpret_cast<RunScale*>(smem + L::kMain) + warp * kStages;
  const uint32_t bars = smem_u32(smem) + L::kMain + L::kScale + warp * kStages * 8;
  const int page_mask = (1 << c.page_shift) - 1;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) mbar_init(bars + 8 * i, 1);
    fence_mbar_init();
  }
  __syncwarp();
  unsigned sent = 0, taken = 0;  // runs that this warp has issued and used, over all parts
  bool alive = true;             // false once a wait ran out: nothing more is issued or used

  for (long long u = u_begin; u < u_end;) {
    SeqWork w = seq_work(c, s, group);
    while (u >= seq_first + w.units(c.Hkv)) {  // on to the sequence of unit u
      if (s + 1 >= c.n_seqs) return;
      seq_first += w.units(c.Hkv);
      w = seq_work(c, ++s, group);
    }
    const long long tuple = (u - seq_first) / w.tiles;
    const int tile0 = static_cast<int>(u - seq_first - tuple * w.tiles);
    const int tile1 = static_cast<int>(min(static_cast<long long>(w.tiles), tile0 + (u_end - u)));
    const int head = static_cast<int>(tuple / w.row_tiles);
    const int row0 = static_cast<int>(tuple - static_cast<long long>(head) * w.row_tiles) * kRows;
    const int rows = min(kRows, w.q.n * group - row0);

    // Rows r and r + 8 of this lane: token, head and number of visible keys.
    int limit[2];
    float row_mul[2];
    uint32_t qf[kSteps][4];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = row0 + r + 8 * x;
      const bool on = r + 8 * x < rows;
      const int token = on ? row / group : 0;
      const int h = head * group + (on ? row - token * group : 0);
      limit[x] = on ? (a.causal ? max(0, w.q.len - w.q.n + token + 1) : w.q.len) : 0;
      const T* src = static_cast<const T*>(a.q) + (w.q.t0 + token) * a.sq[0] + h * a.sq[1];
      // Columns of step t: 4 neighbours, so that a K word is the two halves of a B fragment.
      uint32_t raw[kSteps][2];
#pragma unroll
      for (int p = 0; p < kSteps / 4; ++p) {
        const uint4* at = reinterpret_cast<const uint4*>(src + 16 * k_piece<D>(cq, p));
        const uint4 v0 = on ? __ldg(at) : make_uint4(0, 0, 0, 0);
        const uint4 v1 = on ? __ldg(at + 1) : make_uint4(0, 0, 0, 0);
        const uint32_t f[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[4 * p + i / 2][i & 1] = f[i];
      }
      row_mul[x] = a.scale * kLog2e;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        float big = 0.f;
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 f = to_float2<T>(raw[t][i]);
            big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int e = big > 0.f && big < INFINITY
                          ? min(126, max(-118, static_cast<int>(__float_as_uint(big) >> 23) - 127 - 8))
                          : 0;
        const float div = __int_as_float((127 - e) << 23);
        row_mul[x] *= __int_as_float((127 + e) << 23);
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 f = to_float2<T>(raw[t][i]);
            raw[t][i] = from_float2<__half>(f.x * div, f.y * div);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        qf[t][x] = raw[t][0];
        qf[t][2 + x] = raw[t][1];
      }
    }
    // Keys that the tile's last row sees, and those that all of its rows see.
    const int last_token = (row0 + rows - 1) / group, first_token = row0 / group;
    const int seen = a.causal ? max(0, w.q.len - w.q.n + last_token + 1) : w.q.len;
    const int all_see = a.causal ? max(0, w.q.len - w.q.n + first_token + 1) : w.q.len;

    // Runs of this warp: keys [first_key + i * kTile, + kRun), i < n_runs.
    const int first_key = tile0 * kTile + warp * kRun;
    const int stop = min(seen, tile1 * kTile);
    const int n_runs = first_key < stop ? (stop - first_key + kTile - 1) / kTile : 0;

    // Page numbers and scales of 32 runs at a time, one to a lane, looked up a batch ahead.
    struct Batch {
      int page;
      RunScale sc;
    };
    auto look_up = [&](int i) {
      Batch b;
      b.page = -1;
      b.sc = RunScale{0.f, 0.f, 0.f, 0};
      if (i < n_runs) {
        b.page = page_of(c, s, (first_key + i * kTile) >> c.page_shift);
        if (b.page >= 0) {
          const long long at = static_cast<long long>(b.page) * c.Hkv + head;
          b.sc.mul = __ldg(c.k_scale + at);
          value_scale(__ldg(c.v_scale + at), &b.sc.add, &b.sc.inv);
          b.sc.present = 1;
        }
      }
      return b;
    };
    Batch now = look_up(lane), next = look_up(32 + lane);
    int issued = 0;
    auto issue = [&]() {
      const int i = issued++;
      if (i >= n_runs || !alive) return;
      if (i > 0 && (i & 31) == 0) {
        now = next;
        next = look_up(i + 32 + lane);
      }
      const int stage = sent % kStages;
      ++sent;
      const int page = __shfl_sync(0xffffffffu, now.page, i & 31);
      if (lane == (i & 31)) scales[stage] = now.sc;
      if (lane == 0) {
        const uint32_t bar = bars + 8 * stage, dst = ring + stage * L::kStage;
        if (page >= 0) {
          const int slot = (first_key + i * kTile) & page_mask;
          mbar_arrive_expect_tx(bar, L::kStage);
          load_page(dst, &maps.k, maps.k_pos, slot, head, page, bar);
          load_page(dst + L::kHalf, &maps.v, maps.v_pos, slot, head, page, bar);
        } else {
          mbar_arrive(bar);
        }
      }
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue();

    float acc[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int i = 0; i < n_runs; ++i) {
      const int stage = taken % kStages;
      if (alive) alive = wait_copy(bars + 8 * stage, (taken / kStages) & 1, a);
      alive = __all_sync(0xffffffffu, alive);
      if (!alive) break;
      ++taken;
      issue();  // into the stage that every lane left before the vote
      const uint32_t kb = ring + stage * L::kStage;
      const uint32_t vb = kb + L::kHalf;
      const RunScale sc = scales[stage];

      float sacc[2][2][4] = {};  // [8 keys][even, odd steps]: shorter chains of products
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const int key = nt * 8 + r;
        uint32_t kw[kWords];
#pragma unroll
        for (int p = 0; p < kPieces / 4; ++p) {
          const int piece = k_piece<D>(cq, p);
          const uint4 v = lds128(kb + key * D + (D == 128 ? piece ^ r : piece ^ ((r >> 1) & 3)) * 16);
          kw[4 * p] = v.x, kw[4 * p + 1] = v.y, kw[4 * p + 2] = v.z, kw[4 * p + 3] = v.w;
        }
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
          mma_f16(sacc[nt][t & 1], qf[t], e4m3_lo(kw[t]), e4m3_hi(kw[t]));
        }
      }

      float mul[2] = {sc.mul * row_mul[0], sc.mul * row_mul[1]};
      float t[2][4];  // [row][key]
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          t[e >> 1][nt * 2 + (e & 1)] = fmaf(sacc[nt][0][e] + sacc[nt][1][e], mul[e >> 1], sc.add);
        }
      }
      const int key0 = first_key + i * kTile;
      if (key0 + kRun > all_see || !sc.present) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int lim = sc.present ? limit[x] - key0 : 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if ((e >> 1) * 8 + 2 * cq + (e & 1) >= lim) t[x][e] = -INFINITY;
          }
        }
      }
      float big[2];
      bool moved = false;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        big[x] = fmaxf(fmaxf(t[x][0], t[x][1]), fmaxf(t[x][2], t[x][3]));
        moved |= big[x] > m[x] + kLazy;
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          big[x] = fmaxf(big[x], __shfl_xor_sync(0xffffffffu, big[x], 1));
          big[x] = fmaxf(big[x], __shfl_xor_sync(0xffffffffu, big[x], 2));
          const float to = fmaxf(m[x], big[x]);
          const float f = to == m[x] ? 1.f : ex2_approx(m[x] - to);
          m[x] = to;
          l[x] *= f;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            acc[j][2 * x] *= f;
            acc[j][2 * x + 1] *= f;
          }
        }
      }
      uint32_t pf[4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float ref = m[x] == -INFINITY ? 0.f : m[x];
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = ex2_approx(t[x][e] - ref);
        l[x] = fmaf((p[0] + p[1]) + (p[2] + p[3]), sc.inv, l[x]);
        pf[x] = from_float2<__half>(p[0], p[1]);
        pf[2 + x] = from_float2<__half>(p[2], p[3]);
      }

      // V: this lane's keys 2cq, 2cq + 1, 2cq + 8, 2cq + 9 and columns (D / 8) r .. + D / 8: column
      // block j of the products holds the columns (D / 8) n + j, n = 0..7.
      uint32_t vw[4][D / 32];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int key = 2 * cq + (k & 1) + 8 * (k >> 1);
        if constexpr (D == 128) {
          const uint4 v = lds128(vb + key * D + (r ^ (key & 7)) * 16);
          vw[k][0] = v.x, vw[k][1] = v.y, vw[k][2] = v.z, vw[k][3] = v.w;
        } else {
          const uint2 v = lds64(vb + key * D + ((r >> 1) ^ ((key >> 1) & 3)) * 16 + (r & 1) * 8);
          vw[k][0] = v.x, vw[k][1] = v.y;
        }
      }
      if (key0 + kRun > w.q.len || !sc.present) {  // behind the last key a page holds anything
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (key0 + 2 * cq + (k & 1) + 8 * (k >> 1) >= w.q.len || !sc.present) {
#pragma unroll
            for (int j = 0; j < D / 32; ++j) vw[k][j] = 0;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint32_t a0 = __byte_perm(vw[0][j], vw[1][j], 0x5140);
        const uint32_t a1 = __byte_perm(vw[0][j], vw[1][j], 0x7362);
        const uint32_t b0 = __byte_perm(vw[2][j], vw[3][j], 0x5140);
        const uint32_t b1 = __byte_perm(vw[2][j], vw[3][j], 0x7362);
        mma_f16(acc[4 * j], pf, e4m3_lo(a0), e4m3_lo(b0));
        mma_f16(acc[4 * j + 1], pf, e4m3_hi(a0), e4m3_hi(b0));
        mma_f16(acc[4 * j + 2], pf, e4m3_lo(a1), e4m3_lo(b1));
        mma_f16(acc[4 * j + 3], pf, e4m3_hi(a1), e4m3_hi(b1));
      }
    }
    // Copies in flight when a wait ran out still write to this block's memory.
    while (taken != sent) {
      wait_copy(bars + 8 * (taken % kStages), (taken / kStages) & 1, a);
      ++taken;
    }

    // Merge the warps' sums: each scales its own to the block's maximum, then the block adds.
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (cq == 0) {
        merge_m[warp][r + 8 * x] = m[x];
        merge_l[warp][r + 8 * x] = l[x];
      }
    }
    __syncthreads();  // and no warp reads its ring any more
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float top = merge_m[0][r + 8 * x];
#pragma unroll
      for (int i = 1; i < kWarps; ++i) top = fmaxf(top, merge_m[i][r + 8 * x]);
      const float f = m[x] == -INFINITY ? (l[x] == l[x] ? 0.f : l[x]) : ex2_approx(m[x] - top);
      float* at = sums + (warp * kRows + r + 8 * x) * D;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int j = 0; j < D / 8; j += 4) {
          *reinterpret_cast<float4*>(at + (2 * cq + n) * (D / 8) + j) =
              make_float4(acc[j][2 * x + n] * f, acc[j + 1][2 * x + n] * f,
                          acc[j + 2][2 * x + n] * f, acc[j + 3][2 * x + n] * f);
        }
      }
    }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == w.tiles;
    constexpr int kPer = kRows * D / kThreads;  // columns of one thread
    const int row = tid / (D / kPer), col = (tid % (D / kPer)) * kPer;
    if (row < rows) {
      float top = merge_m[0][row], lsum = 0.f;
#pragma unroll
      for (int i = 1; i < kWarps; ++i) top = fmaxf(top, merge_m[i][row]);
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float wm = merge_m[i][row], wl = merge_l[i][row];
        lsum += wm == -INFINITY ? (wl == wl ? 0.f : wl) : wl * ex2_approx(wm - top);
      }
      float out[kPer];
#pragma unroll
      for (int k = 0; k < kPer; k += 4) {
        float4 v = *reinterpret_cast<const float4*>(sums + row * D + col + k);
#pragma unroll
        for (int i = 1; i < kWarps; ++i) {
          const float4 x = *reinterpret_cast<const float4*>(sums + (i * kRows + row) * D + col + k);
          v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        out[k] = v.x, out[k + 1] = v.y, out[k + 2] = v.z, out[k + 3] = v.w;
      }
      if (whole) {
        const int token = (row0 + row) / group;
        const long long at = static_cast<long long>(w.q.t0 + token) * a.H + head * group +
                             (row0 + row - token * group);
        const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
        T* o = static_cast<T*>(a.o) + at * D + col;
#pragma unroll
        for (int k = 0; k < kPer; k += 8) {
          uint4 v;
          v.x = from_float2<T>(out[k] * inv, out[k + 1] * inv);
          v.y = from_float2<T>(out[k + 2] * inv, out[k + 3] * inv);
          v.z = from_float2<T>(out[k + 4] * inv, out[k + 5] * inv);
          v.w = from_float2<T>(out[k + 6] * inv, out[k + 7] * inv);
          *reinterpret_cast<uint4*>(o + k) = v;
        }
        if (col == 0) a.lse[at] = lsum == 0.f ? INFINITY : (top + log2f(lsum)) * kLn2;
      } else {
        float* part = partials + (2ll * blockIdx.x + (u == u_begin ? 0 : 1)) * partial_floats(D);
#pragma unroll
        for (int k = 0; k < kPer; k += 4) {
          *reinterpret_cast<float4*>(part + row * D + col + k) =
              make_float4(out[k], out[k + 1], out[k + 2], out[k + 3]);
        }
        if (col == 0) {
          part[kRows * D + row] = top;
          part[kRows * D + kRows + row] = lsum;
        }
      }
    }
    fence_proxy_async_smem();  // the sums were read: the next part's copies may overwrite them
    __syncthreads();
    u += tile1 - tile0;
  }
}

// Merges the parts of a tuple that several CTAs share.  Block i looks after the tuple that CTA i's
// range begins inside of, if no earlier CTA's does too.  Each row's parts are split over warps.
constexpr int kCombineWarps = 16;

template <typename T, int D>
__global__ void __launch_bounds__(32 * kCombineWarps) fa_cache_combine_kernel(
    const __grid_constant__ CacheAttnArgs a, const float* partials) {
  constexpr int kPer = D / 32;
  __shared__ Finder<32 * kCombineWarps> finder;
  __shared__ float sums[kCombineWarps][D];
  __shared__ float tops[kCombineWarps], lsums[kCombineWarps];
  const CacheView& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = a.H / c.Hkv;
  const int me = blockIdx.x;
  const long long total = finder.total(c, group);
  const int ctas = ctas_of(total);
  if (me == 0 || me >= ctas) return;
  const long long begin = bound_of(total, me, ctas);
  finder.find(c, group, begin);
  const int s = finder.at.s;
  const long long seq_first = finder.at.first;
  const SeqWork w = seq_work(c, s, group);
  const long long tuple = (begin - seq_first) / w.tiles;
  const long long first = seq_first + tuple * w.tiles, end = first + w.tiles;
  if (first == begin || bound_of(total, me - 1, ctas) > first) return;
  const int head = static_cast<int>(tuple / w.row_tiles);
  const int row0 = static_cast<int>(tuple - static_cast<long long>(head) * w.row_tiles) * kRows;
  const int rows = min(kRows, w.q.n * group - row0);
  asm volatile("griddepcontrol.wait;" ::: "memory");

  int split = 1;  // rows side by side; the warps of a row share its parts
  while (split < rows) split *= 2;
  const int row = warp % split, share = warp / split, shares = kCombineWarps / split;
  int last = me;  // one past the last CTA with a part
  while (last < ctas && bound_of(total, last, ctas) < end) ++last;
  float top = -INFINITY, lsum = 0.f, acc[kPer] = {};
  if (row < rows) {
    for (int i = me - 1 + share; i < last; i += shares) {
      const int slot = bound_of(total, i, ctas) >= first ? 0 : 1;
      const float* part = partials + (2ll * i + slot) * partial_floats(D);
      const float pm = part[kRows * D + row], pl = part[kRows * D + kRows + row];
      if (pm == -INFINITY && pl == 0.f) continue;
      float v[kPer];
#pragma unroll
      for (int k = 0; k < kPer; ++k) v[k] = part[row * D + lane * kPer + k];
      const float to = fmaxf(top, pm);
      const float f0 = top == -INFINITY ? 0.f : ex2_approx(top - to);
      const float f1 = pm == -INFINITY ? 1.f : ex2_approx(pm - to);
      top = to;
      lsum = lsum * f0 + pl * f1;
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[k] = acc[k] * f0 + v[k] * f1;
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) sums[warp][lane * kPer + k] = acc[k];
  if (lane == 0) {
    tops[warp] = top;
    lsums[warp] = lsum;
  }
  __syncthreads();
  if (share > 0 || row >= rows) return;
  for (int i = 1; i < shares; ++i) {
    const int other = row + i * split;
    const float pm = tops[other], pl = lsums[other];
    if (pm == -INFINITY && pl == 0.f) continue;
    const float to = fmaxf(top, pm);
    const float f0 = top == -INFINITY ? 0.f : ex2_approx(top - to);
    const float f1 = pm == -INFINITY ? 1.f : ex2_approx(pm - to);
    top = to;
    lsum = lsum * f0 + pl * f1;
#pragma unroll
    for (int k = 0; k < kPer; ++k) acc[k] = acc[k] * f0 + sums[other][lane * kPer + k] * f1;
  }
  const int token = (row0 + row) / group;
  const long long at = static_cast<long long>(w.q.t0 + token) * a.H + head * group +
                       (row0 + row - token * group);
  const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
  uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<T*>(a.o) + at * D + lane * kPer);
#pragma unroll
  for (int k = 0; k < kPer; k += 2) o[k / 2] = from_float2<T>(acc[k] * inv, acc[k + 1] * inv);
  if (lane == 0) a.lse[at] = lsum == 0.f ? INFINITY : (top + log2f(lsum)) * kLn2;
}

int decode_ctas(int sms) { return kPerSm * sms; }

template <typename T, int D>
cudaError_t launch_t(const CacheAttnArgs& a, cudaStream_t stream) {
  const CacheView& c = a.c;
  const int group = a.H / c.Hkv;
  // No more CTAs than units that the table could hold.
  const long long room = static_cast<long long>(c.max_pages) << c.page_shift;
  const long long tiles = std::max(1ll, (room + kTile - 1) / kTile);
  const long long tuples =
      (static_cast<long long>(c.T) * group / kRows + c.n_seqs) * c.Hkv;
  const long long want = std::min<long long>(decode_ctas(multiprocessors()),
                                             tuples > (1ll << 40) / tiles ? (1ll << 40) : tuples * tiles);
  const unsigned ctas = static_cast<unsigned>(std::max(1ll, want));
  float* partials = static_cast<float*>(a.workspace);
  constexpr int kSmem = Layout<D>::kBytes;
  PageMaps maps;
  cudaError_t e = make_page_maps(&maps, c, D, kRun);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(fa_cache_decode_kernel<T, D>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  fa_cache_decode_kernel<T, D><<<ctas, kThreads, kSmem, stream>>>(a, maps, partials);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if (tiles == 1) return cudaSuccess;  // no tuple has two units
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(32 * kCombineWarps);
  cfg.stream = stream;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fa_cache_combine_kernel<T, D>, a,
                            static_cast<const float*>(partials));
}

}  // namespace

size_t cache_attention_workspace(int, int, int D, int, int, int sms) {
  return 2ull * decode_ctas(sms) * partial_floats(D) * sizeof(float);
}

cudaError_t launch_cache_attention(const CacheAttnArgs& a, cudaStream_t stream) {
  if (a.dtype == FA_DTYPE_F16) {
    return a.D == 64 ? launch_t<__half, 64>(a, stream) : launch_t<__half, 128>(a, stream);
  }
  return a.D == 64 ? launch_t<__nv_bfloat16, 64>(a, stream)
                   : launch_t<__nv_bfloat16, 128>(a, stream);
}

}  // namespace fa_sm100
