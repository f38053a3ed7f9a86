// fa_cache_tile.cu -- attention over the paged e4m3 cache for sequences with many query rows: prompt
// chunks, drafts, mixed batches.  Same mathematics as fa_cache_attn.cu (see there); here the two
// products run on tcgen05 with their accumulators in tensor memory.
//
// A tile is up to 256 query rows of one (sequence, kv head): rows are (token, head of the group)
// packed, so the group's heads share every key that is loaded and converted.  Keys come 128 at a time
// (one unit of work).  The units of all sequences are numbered and split evenly over one CTA for each
// multiprocessor; a tile that several CTAs share leaves fp32 partials for fa_cache_tile_merge_kernel.
//
//   warp 16      looks pages and scales up
//   warps 8-11   (K) and 12-15 (V) load e4m3 pages into registers, a tile ahead, and store them as
//                fp16 in the swizzled layout of the products (exact; two buffers each): tcgen05 has
//                no product of fp16 by e4m3, and rounding q and P to 8 bits would cost what the
//                cache's own 8 bits cost again.  Registers and not TMA: a tile in flight takes no
//                shared memory, which the fp16 buffers fill.  (With e4m3 tiles in shared memory V had
//                one buffer, and its conversion, 1100 cycles, stood between two products.)
//   warps 17, 18 issue S = Q K^T and O += P V of a group each
//   warps 0-3, 4-7   two softmax groups, a row to a thread.  With more than 128 rows group g has rows
//                128 g .. and every key tile; otherwise both have the same rows and the key tiles
//                alternate, and their sums are merged at the end (both lie in one lane of tensor
//                memory).  Either way the tensor core works for one group while the other
//                exponentiates.
//
// A key tile goes through in two halves of 64 keys: S_g has two buffers of 64 columns in tensor memory,
// P_g (fp16) overwrites the first 32 of its own, O_g takes D.  While a group exponentiates one half
// the products of the other are under way.
//
// What bounds it: 2048 new tokens of 32 heads over 16384 keys of 8 heads of 128 take 644 us, 800 TFLOP/s,
// about 4700 cycles for 256 rows by 128 keys where the products alone need 2048.  A group's softmax of
// 64 keys takes 2250 cycles (maximum 500, exponentials 1000, the rest loads, stores and hand-offs), and
// the products, S reading both operands from shared memory and sharing it with the conversion's stores,
// 3400 of the 4700.  8 sequences of 1 to 801 new tokens over 300 to 6001 keys of 4 heads take 157 us, where a
// change of tile, 24000 cycles from product to product instead of 4700, weighs most: a CTA has 26 units of 2.1
// tiles on average and of 7 at most, and units alone are dealt evenly.
//
// Measured and not kept: four softmax groups with a row's maximum handed from half to half (650 us), a
// quarter of the exponentials as polynomials on the FMA pipes (638 us), products issued by one lane of a
// diverged warp (738 us: operands have to move to uniform registers one by one).  One S of 128 columns, one
// warp for all products and one group of warps that converts K and V by way of e4m3 tiles in shared memory took
// 611 us for the first of these calls on the GPU of the 644, and 184 for the second where this takes 156; with S
// in halves and conversion through registers, 614 and 165.  Of the 33 us, 10 go into taking V's NaN out of
// the tiles on the diagonal.
#include <algorithm>
#include <cmath>

#include "fa_cache_common.cuh"
#include "sm100_ptx.cuh"

namespace fa_sm100 {
namespace {

constexpr int kThreads = 640;
constexpr int kRows = 256;   // query rows of a tile
constexpr int kHalfRows = 128;
constexpr int kKeys = 128;   // keys of a unit
constexpr int kGroups = kKeys / 16;
constexpr int kTables = 8;   // scale tables in flight: more than the tiles between load and softmax
constexpr int kPairBarrier = 1;  // named barrier of the two softmax groups
constexpr float kLazy = 8.0f;
constexpr float kSmallest = 1.1754944e-38f;  // a factor that -inf times is -inf
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct Layout {
  static constexpr int kChunks = D / 64;             // 128-byte column chunks of an fp16 tile
  static constexpr int kChunkBytes = kKeys * 128;
  static constexpr int kTile16 = kChunks * kChunkBytes;  // 128 rows of fp16 (Q half, K or V tile)
  static constexpr int kQ = 0;
  static constexpr int kK16 = kQ + 2 * kTile16;
  static constexpr int kV16 = kK16 + 2 * kTile16;
  static constexpr int kTable = kV16 + 2 * kTile16;
  static constexpr int kBars = kTable + kTables * kGroups * 32;
  // Barriers.
  // kSFull, kPFull: group g, half h at + 2 g + h.
  static constexpr int kK16Full = 0, kK16Empty = 2, kV16Full = 4, kV16Empty = 6, kSFull = 8,
                       kPFull = 12, kODone = 16, kOFull = 18, kQFull = 20, kTabFull = 22,
                       kTabEmpty = kTabFull + kTables, kDrain = kTabEmpty + kTables,
                       kCount = kDrain + 1;
  static constexpr int kMisc = kBars + 8 * kCount;
  static constexpr int kClean = kMisc + 16;  // per table: every key of the tile is there
  static constexpr int kBytes = kClean + 4 * kTables + 1024;
  static constexpr int kColS = 0, kColO = 256, kCols = 512;
  static constexpr int kPartial = kRows * D + 2 * kRows;  // floats
  static_assert(kBytes <= 230000, "shared memory overflow");  // and some for the static part
};

// 16 keys: what their scores need, and where they lie.
struct RunScale {
  float mul, add, inv;
  int page;
  long long k_at, v_at;  // byte offsets of the first key
};

// ---- work ----

// sum over i < n of floor((2 i + b) / m)
__device__ __forceinline__ long long sum_floors(unsigned n, unsigned m, unsigned b) {
  long long sum = 0;
  unsigned a = 2;
  for (;;) {
    if (a >= m) {
      sum += static_cast<long long>(n) * (n - 1ll) / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      sum += static_cast<long long>(n) * (b / m);
      b %= m;
    }
    const unsigned y = a * n + b;
    if (y < m) return sum;
    n = y / m;
    b = y % m;
    const unsigned t = m;
    m = a;
    a = t;
  }
}

// The tiles of one (sequence, kv head).  With past = len - n, which is negative where queries lie in front
// of the keys, tile j's last row is a query that sees past + floor((256 j + 255) / group) + 1 keys (causal),
// so the tile has max(1, floor((2 j + base) / group)) units, base = floor((255 + group (past + 128)) / 128):
// one in each of the first `flat` tiles, and behind them a sum with a closed form.  The last tile ends
// with the last row, which sees every key; no tile has more units than the keys make.
struct SeqTiles {
  SeqInfo q;
  int rows, tiles;
  bool causal;
  int full;        // units of the last tile; not causal: of each
  int flat;        // causal: tiles in front that see at most one unit's keys ...
  long long base;  // ... see above
  long long units;  // of one kv head

  __device__ long long before(int j, int group) const {
    if (!causal) return static_cast<long long>(j) * full;
    if (j <= flat) return j;
    const long long at = base + 2ll * flat, whole = at / group;
    return flat + whole * (j - flat) + sum_floors(j - flat, group, static_cast<unsigned>(at - whole * group));
  }
  __device__ int of(int j, int group) const {
    if (j == tiles - 1 || !causal) return full;
    return j < flat ? 1 : static_cast<int>((2ll * j + base) / group);
  }
};

__device__ __forceinline__ SeqTiles tiles_of(const SeqInfo& q, int group, bool causal) {
  SeqTiles t;
  t.q = q;
  t.causal = causal;
  t.rows = q.n * group;
  t.tiles = (t.rows + kRows - 1) / kRows;
  t.full = max(1, (q.len + kKeys - 1) / kKeys);
  t.flat = 0;
  t.base = 0;
  t.units = 0;
  if (t.tiles == 0) return t;
  if (causal) {
    t.base = (255 + group * (static_cast<long long>(q.len) - q.n + kKeys)) >> 7;
    static_assert(kKeys == 1 << 7, "floors of negative numbers by shifts");
    t.flat = static_cast<int>(min(static_cast<long long>(t.tiles), max(0ll, (group - t.base + 1) >> 1)));
  }
  t.units = t.before(t.tiles - 1, group) + t.full;
  return t;
}

__device__ __forceinline__ long long units_per_cta(long long total) {
  return (total + gridDim.x - 1) / gridDim.x;
}

// A place in the list of units: unit `u` is unit `tile` of row tile `j` of kv head `head`.
struct Place {
  int s, head, j, tile;
};

// All CTAs add up the units of the sequences and find the place that their own range begins at.
template <int THREADS>
struct Finder {
  long long warp[THREADS / 32];
  SeqInfo q;
  long long first;
  Place at;

  __device__ long long scan(long long x, long long* sum) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += up;
    }
    __syncthreads();
    if (lane == 31) warp[wid] = x;
    __syncthreads();
    *sum = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < wid) x += warp[i];
      *sum += warp[i];
    }
    return x;
  }

  // Returns the total of units; places the first unit of CTA `cta`'s range, if it has one.
  __device__ long long find(const CacheView& c, int group, bool causal, int cta, long long* per) {
    if (threadIdx.x == 0) {
      at = Place{0, 0, 0, 0};
      q = SeqInfo{0, 0, 0};
      first = 0;
    }
    long long mine = 0, incl = 0, total = 0, sum;
    for (int base = 0; base < c.n_seqs; base += THREADS) {
      const int s = base + threadIdx.x;
      mine = s < c.n_seqs ? tiles_of(seq_info(c, s), group, causal).units * c.Hkv : 0;
      incl = total + scan(mine, &sum);
      total += sum;
    }
    *per = units_per_cta(total);
    const long long unit = cta * *per;
    if (unit < total) {
      long long run = 0;
      for (int base = 0; base < c.n_seqs; base += THREADS) {
        const int s = base + threadIdx.x;
        if (c.n_seqs > THREADS) {
          mine = s < c.n_seqs ? tiles_of(seq_info(c, s), group, causal).units * c.Hkv : 0;
          incl = run + scan(mine, &sum);
          run += sum;
        }
        if (mine > 0 && unit < incl && unit >= incl - mine) {
          at.s = s;
          q = seq_info(c, s);
          first = incl - mine;
        }
      }
      __syncthreads();
      if (threadIdx.x < 32) {  // 32 probes at a time for the row tile
        const SeqTiles t = tiles_of(q, group, causal);
        long long rel = unit - first;
        const int head = t.units > 0 ? static_cast<int>(rel / t.units) : 0;
        rel -= head * t.units;
        int lo = 0, n = t.tiles;
        while (n > 1) {
          const int step = (n + 31) / 32;
          const int probe = static_cast<int>(threadIdx.x) * step;
          const bool below = probe < n && t.before(lo + probe, group) <= rel;
          const int hit = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
          lo += hit * step;
          n = min(step, n - hit * step);
        }
        if (threadIdx.x == 0) {
          at.head = head;
          at.j = lo;
          at.tile = static_cast<int>(rel - t.before(lo, group));
        }
      }
    }
    __syncthreads();
    return total;
  }
};

// The part of a tile that a CTA works on.  Every warp walks the parts by itself, in shared memory:
// they change seldom, and registers are short.
struct Part {
  SeqTiles t;
  Place p;
  long long left;  // units of the CTA's range from here on
  int row0, rows;
  int tile0, tile1;  // its units
  int n_tiles;       // those that hold keys that a row sees
  int seen;          // keys that the last row sees
  bool pair;         // at most 128 rows: the key tiles alternate between the groups
  bool whole;
  bool more;         // false behind the last part

  template <int THREADS>
  __device__ void start(const Finder<THREADS>& f, int group, bool causal, long long units) {
    t = tiles_of(f.q, group, causal);
    p = f.at;
    left = units;
    more = true;
    set(group);
  }
  __device__ void set(int group) {
    const int units = t.of(p.j, group);
    row0 = p.j * kRows;
    rows = min(kRows, t.rows - row0);
    tile0 = p.tile;
    tile1 = static_cast<int>(min(static_cast<long long>(units), tile0 + left));
    whole = tile0 == 0 && tile1 == units;
    const int last_token = (row0 + rows - 1) / group;
    seen = t.causal ? min(t.q.len, max(0, t.q.len - t.q.n + last_token + 1)) : t.q.len;
    n_tiles = max(0, min(tile1, (seen + kKeys - 1) / kKeys) - tile0);
    pair = rows <= kHalfRows;
  }
  // On to the next part; `more` is false at the end of the range.
  __device__ void next(const CacheView& c, int group) {
    left -= tile1 - tile0;
    more = false;
    if (left <= 0) return;
    p.tile = 0;
    if (++p.j >= t.tiles) {
      p.j = 0;
      if (++p.head >= c.Hkv) {
        p.head = 0;
        do {
          if (++p.s >= c.n_seqs) return;
          t = tiles_of(seq_info(c, p.s), group, t.causal);
        } while (t.tiles == 0);
      }
    }
    more = true;
    set(group);
  }
};

// ---- waits ----

struct Waits {
  volatile int* abort_flag;
  unsigned long long timeout_ns;
  unsigned* status;
};

__device__ __forceinline__ bool wait_or_abort(uint32_t bar, uint32_t parity, const Waits& w,
                                              unsigned cause) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (;;) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*w.abort_flag) return false;
    if (globaltimer_ns() - t0 > w.timeout_ns) {
      *w.abort_flag = 1;
      atomicOr(w.status, cause);
      return false;
    }
  }
}

// For this CTA's own copies and products in flight, on the way out.
__device__ __forceinline__ void wait_out(uint32_t bar, uint32_t parity, const Waits& w) {
  if (mbar_try_wait(bar, parity)) return;
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > max(w.timeout_ns, kMinDrainNs)) {
      atomicOr(w.status, kStDrain);
      return;
    }
  }
}

// ---- pieces of the roles ----

// 16 bytes that are read once by this block.
__device__ __forceinline__ uint4 ldg128(const unsigned char* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// Four e4m3 values as two words of fp16.
__device__ __forceinline__ uint2 widen(uint32_t u) {
  uint2 r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(r.x), "=r"(r.y)
      : "r"(u));
  return r;
}

// 16 e4m3 values as fp16, 16 bytes at `lo` and 16 at `hi`.
__device__ __forceinline__ void store_wide(uint32_t lo, uint32_t hi, uint4 v) {
  const uint2 a = widen(v.x), b = widen(v.y), c = widen(v.z), d = widen(v.w);
  sts128(lo, make_uint4(a.x, a.y, b.x, b.y));
  sts128(hi, make_uint4(c.x, c.y, d.x, d.y));
}

// The larger one, NaN where one is NaN.
__device__ __forceinline__ float fmax_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// True in one lane of the (converged) warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// The 256 threads of the two softmax groups.
__device__ __forceinline__ void pair_barrier() {
  asm volatile("bar.sync %0, 256;" ::"n"(kPairBarrier) : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) fa_cache_tile_kernel(
    const __grid_constant__ CacheAttnArgs a, float* partials) {
  using L = Layout<D>;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (sbase - raw);
  __shared__ Finder<kThreads> finder;
  __shared__ Part parts[kThreads / 32];
  RunScale* tables = reinterpret_cast<RunScale*>(smem + L::kTable);
  volatile int* clean = reinterpret_cast<volatile int*>(smem + L::kClean);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  // One more than the last tile that NaN were taken out of V of (see nan_columns).
  unsigned* last_nan = reinterpret_cast<unsigned*>(smem + L::kMisc + 8);
  auto bar = [sbase](int i) -> uint32_t { return sbase + L::kBars + 8u * i; };
  const CacheView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = a.H / c.Hkv;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  zero_stray_rows<T, D, kThreads>(a);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(L::kK16Full + i), 4);
      mbar_init(bar(L::kK16Empty + i), 2);
      mbar_init(bar(L::kV16Full + i), 4);
      mbar_init(bar(L::kV16Empty + i), 2);
      mbar_init(bar(L::kODone + i), 1);
      mbar_init(bar(L::kOFull + i), 1);
      mbar_init(bar(L::kQFull + i), kHalfRows);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(L::kSFull + i), 1);
      mbar_init(bar(L::kPFull + i), kHalfRows);
    }
    for (int i = 0; i < kTables; ++i) {
      mbar_init(bar(L::kTabFull + i), 1);
      mbar_init(bar(L::kTabEmpty + i), 2);
    }
    mbar_init(bar(L::kDrain), 2);
    *abort_flag = 0;
    *last_nan = 0;
    fence_mbar_init();
  }
  long long per;
  const long long total = finder.find(c, group, a.causal, blockIdx.x, &per);
  const long long u_begin = blockIdx.x * per;
  if (u_begin >= total) return;  // the whole block
  const long long n_units = min(total - u_begin, per);
  if (warp == 17) {
    tmem_alloc(smem_u32(tmem_slot), L::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Waits w{abort_flag, a.timeout_ns, c.status};
  Part& part = parts[warp];
  if (lane == 0) part.start(finder, group, a.causal, n_units);
  __syncwarp();
  auto next_part = [&]() {  // by whole warps
    __syncwarp();
    if (lane == 0) part.next(c, group);
    __syncwarp();
    return part.more;
  };

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax groups
    regs_alloc<136>();  // 256 x 136 + 256 x 72 + 128 x 64 = 640 x 96
    const int g = warp >> 2;
    const int r = tid & 127;  // tensor-memory lane
    const uint32_t tl = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_col = tl + L::kColS + g * 128, o_col = tl + L::kColO + g * 128;
    unsigned steps_done = 0, tiles_done = 0, parts_done = 0;
    bool ok = true;
    bool first_part = true;
    do {
      const SeqInfo q = part.t.q;
      const int row = part.pair ? r : g * kHalfRows + r;
      const bool on = row < part.rows;
      const int token = on ? (part.row0 + row) / group : 0;
      const int h = part.p.head * group + (on ? part.row0 + row - token * group : 0);
      const int limit = on ? (a.causal ? max(0, q.len - q.n + token + 1) : q.len) : 0;
      const int my_steps = 2 * (part.pair ? (part.n_tiles - g + 1) / 2 : part.n_tiles);  // halves
      float row_mul = a.scale * kLog2e;
      float m = -INFINITY, l = 0.f;
      if (part.n_tiles > 0 && ok) {
        // The warp's 32 rows of Q as fp16, swizzled: neighbouring lanes have neighbouring 16 bytes of a
        // row (a row to a thread touched 32 lines with every load), all loads first.
        constexpr int kLanes = D / 8, kRowsAtOnce = 32 / kLanes;
        const int sub = lane / kLanes, piece = lane % kLanes;
        const int r0 = (warp & 3) * 32 + sub;
        const int row1 = part.pair ? r0 : g * kHalfRows + r0;
        int token1 = (part.row0 + row1) / group;
        int h1 = part.row0 + row1 - token1 * group;
        const int rows_left = part.rows - row1;
        const T* const q0 = static_cast<const T*>(a.q) + static_cast<long long>(q.t0) * a.sq[0] +
                            static_cast<long long>(part.p.head) * group * a.sq[1] + piece * 8;
        uint4 v[kLanes];
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
          v[i] = make_uint4(0, 0, 0, 0);
          if (i * kRowsAtOnce < rows_left) {
            v[i] = __ldg(reinterpret_cast<const uint4*>(q0 + token1 * a.sq[0] + h1 * a.sq[1]));
          }
          for (h1 += kRowsAtOnce; h1 >= group; h1 -= group) ++token1;
        }
        int e_own = 0;
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
          const int r1 = r0 + i * kRowsAtOnce;
          if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            uint32_t big = __vmaxu2(__vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu),
                                    __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu));
#pragma unroll
            for (int o = kLanes / 2; o > 0; o /= 2) {
              big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, o));
            }
            const uint32_t top = max(big & 0xffffu, big >> 16);  // infinities and NaN: no division
            const int e = top > 0 && top < 0x7f80u
                              ? min(119, max(-118, static_cast<int>(top >> 7) - 127 - 8)) : 0;
            const float div = __int_as_float((127 - e) << 23);
            uint32_t* u = reinterpret_cast<uint32_t*>(&v[i]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = to_float2<T>(u[k]);
              u[k] = from_float2<__half>(f.x * div, f.y * div);
            }
            const int got = __shfl_sync(0xffffffffu, e, (lane % kRowsAtOnce) * kLanes);
            if (lane / kRowsAtOnce == i) e_own = got;
          }
          if (!part.pair || g == 0) {
            sts128(sbase + L::kQ + g * L::kTile16 + r1 * 128 + (piece >> 3) * L::kChunkBytes +
                       (((piece & 7) ^ (r1 & 7)) * 16),
                   v[i]);
          }
        }
        row_mul *= __int_as_float((127 + e_own) << 23);
        if (!part.pair || g == 0) {
          fence_proxy_async_smem();
          mbar_arrive(bar(L::kQFull + g));
        }
      }
      // The first key that some row of this half does not see.
      const int first_row = part.pair ? 0 : min(g * kHalfRows, part.rows - 1);
      const int all_see = a.causal ? q.len - q.n + (part.row0 + first_row) / group + 1 : q.len;
      for (int k = 0; k < my_steps && ok; ++k) {
        const int half = k & 1, i = part.pair ? 2 * (k >> 1) + g : k >> 1;
        const unsigned at = tiles_done + i;
        const int slot = at % kTables;
        const RunScale* table = tables + slot * kGroups + half * (kGroups / 2);
        if (half == 0) ok = wait_or_abort(bar(L::kTabFull + slot), (at / kTables) & 1, w, kStKFull);
        float mul[kGroups / 2], add[kGroups / 2], inv[kGroups / 2];
        if (ok) {
#pragma unroll
          for (int x = 0; x < kGroups / 2; ++x) {
            const float4 sc = *reinterpret_cast<const float4*>(&table[x]);
            mul[x] = fmax_nan(sc.x * row_mul, kSmallest);
            add[x] = sc.y;
            inv[x] = sc.z;
          }
          ok = wait_or_abort(bar(L::kSFull + 2 * g + half), (steps_done >> 1) & 1, w, kStSFull);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t col0 = s_col + 64 * half;
        const int key0 = (part.tile0 + i) * kKeys + 64 * half;
        uint32_t u[64];
        tmem_ld64_wait(col0, u);
        if (key0 + 64 > all_see || !clean[slot]) {
          const int lim = limit - key0;
#pragma unroll
          for (int x = 0; x < kGroups / 2; ++x) {
            const int lx = table[x].page < 0 ? 0 : lim;
            if (16 * x >= lx) {  // the page's scales are not this row's, and may be NaN
              mul[x] = kSmallest;
              add[x] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              if (16 * x + j >= lx) u[16 * x + j] = 0xff800000u;  // -inf
            }
          }
        }
        float top = m;
#pragma unroll
        for (int x = 0; x < kGroups / 2; ++x) {
          float b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            b[j] = fmaxf(__uint_as_float(u[16 * x + 4 * j]), __uint_as_float(u[16 * x + 4 * j + 1]));
            b[j] = fmax3(b[j], __uint_as_float(u[16 * x + 4 * j + 2]),
                         __uint_as_float(u[16 * x + 4 * j + 3]));
          }
          top = fmaxf(top, fmaf(fmax3(b[0], b[1], fmaxf(b[2], b[3])), mul[x], add[x]));
        }
        const bool moved = top > m + kLazy || (m == -INFINITY && top != -INFINITY);
        const float alpha = moved ? (m == -INFINITY ? 0.f : ex2_approx(m - top)) : 1.f;
        if (moved) m = top;
        const float ref = m == -INFINITY ? 0.f : m;
        l *= alpha;
#pragma unroll
        for (int x = 0; x < kGroups / 2; x += 2) {
          uint32_t pk[16];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint64_t mul2 = f2_pack(mul[x + y], mul[x + y]);
            const uint64_t add2 = f2_pack(add[x + y] - ref, add[x + y] - ref);
            uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int at2 = 16 * (x + y) + 2 * j;
              const uint64_t z =
                  f2_fma(f2_pack(__uint_as_float(u[at2]), __uint_as_float(u[at2 + 1])), mul2, add2);
              const float p0 = ex2_approx(f2_lo(z)), p1 = ex2_approx(f2_hi(z));
              pk[8 * y + j] = pack2<__half>(p0, p1);
              sum[j & 1] = f2_add(sum[j & 1], f2_pack(p0, p1));
            }
            const uint64_t both = f2_add(sum[0], sum[1]);
            l = fmaf(f2_lo(both) + f2_hi(both), inv[x + y], l);
          }
          tmem_st16(col0 + 8 * x, pk);
        }
        tmem_st_wait();
        if (k > 0 && __any_sync(0xffffffffu, moved)) {
          // O follows the maximum once the step before has been added to it.  The barrier counts this
          // group's steps: it cannot pass this one, whose P is still to come, and has passed the last
          // but one, which this step's S comes after.
          ok = __all_sync(0xffffffffu, wait_or_abort(bar(L::kODone + g), (steps_done - 1) & 1, w, kStODone));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int col = 0; col < D; col += 32) {
            uint32_t o[32];
            tmem_ld32_wait(o_col + col, o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
            tmem_st32(o_col + col, o);
          }
          tmem_st_wait();
        }
        ++steps_done;
        tc_fence_before();
        mbar_arrive(bar(L::kPFull + 2 * g + half));
      }
      const unsigned first_tile = tiles_done;
      tiles_done += part.n_tiles;
      if (my_steps > 0 && ok) {
        // A barrier of its own: of the last two steps' phases of kODone either may be the current one.
        ok = wait_or_abort(bar(L::kOFull + g), parts_done & 1, w, kStODone);
        ++parts_done;
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      // Alternating tiles: group 0 merges.  Both groups' sums of a row are in one lane of tensor
      // memory; (m, l) of group 1 go there too, over its scores.  Both groups come to each of these
      // barriers, whatever went wrong.
      const bool merge = part.pair && part.n_tiles > 1;
      float m1 = -INFINITY, l1 = 0.f;
      if (merge) {
        if (g == 1) {
          const uint32_t ml[8] = {__float_as_uint(m), __float_as_uint(l), 0, 0, 0, 0, 0, 0};
          tmem_st8(s_col, ml);
          tmem_st_wait();
          tc_fence_before();
        }
        pair_barrier();
        if (g == 0) {
          tc_fence_after();
          uint32_t ml[32];
          tmem_ld32_wait(tl + L::kColS + 128, ml);
          m1 = __uint_as_float(ml[0]);
          l1 = __uint_as_float(ml[1]);
        }
      }
      // Tensor-memory loads are by the warp: rows that are off take part and store nothing.
      if (ok && (!part.pair || g == 0)) {
        const float top = fmaxf(m, m1);
        const float f0 = m == -INFINITY ? 0.f : ex2_approx(m - top);
        const float f1 = m1 == -INFINITY ? 0.f : ex2_approx(m1 - top);
        // A row whose scores are all NaN has no maximum but a sum that is NaN.
        const float lsum = (m == -INFINITY ? l : l * f0) + (m1 == -INFINITY ? l1 : l1 * f1);
        const float w0 = lsum != lsum ? lsum : f0, w1 = lsum != lsum ? lsum : f1;
        const float inv = part.whole ? (lsum == 0.f ? 0.f : 1.f / lsum) : 1.f;
        const long long at = static_cast<long long>(q.t0 + token) * a.H + h;
        float* slot = partials + (2ll * blockIdx.x + (first_part ? 0 : 1)) * L::kPartial;
        const uint32_t stage = sbase + L::kQ + g * L::kTile16 + (warp & 3) * 4096;
        // A later part's tiles may be counted already: then the search finds nothing.
        const bool spoiled = *reinterpret_cast<volatile unsigned*>(last_nan) > first_tile;
#pragma unroll 1
        for (int col = 0; col < D; col += 32) {
          uint32_t u[32];
          __syncwarp();
          if (my_steps > 0) {
            tmem_ld32_wait(o_col + col, u);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] = 0;
          }
          float o[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __uint_as_float(u[j]) * w0;
          if (merge) {
            tmem_ld32_wait(o_col + 128 + col, u);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = fmaf(__uint_as_float(u[j]), w1, o[j]);
          }
          if (spoiled && part.n_tiles > 0) {
            const int diag = max(0, q.len - q.n + part.row0 / group + 1) & ~(kKeys - 1);
            const uint32_t bits = nan_columns<32>(
                c, part.p.s, part.p.head, max(part.tile0 * kKeys, diag),
                min(limit, (part.tile0 + part.n_tiles) * kKeys), col);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (bits >> j & 1) o[j] = __int_as_float(0x7fffffff);
            }
          }
          // Through shared memory (Q's, which every S has read), so that neighbouring lanes store
          // neighbouring 16 bytes of a row.
          if (part.whole) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint4 x;
              x.x = from_float2<T>(o[8 * j] * inv, o[8 * j + 1] * inv);
              x.y = from_float2<T>(o[8 * j + 2] * inv, o[8 * j + 3] * inv);
              x.z = from_float2<T>(o[8 * j + 4] * inv, o[8 * j + 5] * inv);
              x.w = from_float2<T>(o[8 * j + 6] * inv, o[8 * j + 7] * inv);
              sts128(stage + lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16), x);
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r1 = 8 * i + (lane >> 2), piece = lane & 3;
              const uint4 x = lds128(stage + r1 * 64 + ((piece ^ ((r1 >> 1) & 3)) * 16));
              const long long at1 = __shfl_sync(0xffffffffu, at, r1);
              if (row - lane + r1 < part.rows) {
                *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + at1 * D + col + 8 * piece) = x;
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              sts128(stage + lane * 128 + ((j ^ (lane & 7)) * 16),
                     make_uint4(__float_as_uint(o[4 * j]), __float_as_uint(o[4 * j + 1]),
                                __float_as_uint(o[4 * j + 2]), __float_as_uint(o[4 * j + 3])));
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r1 = 4 * i + (lane >> 3), piece = lane & 7;
              const uint4 x = lds128(stage + r1 * 128 + ((piece ^ (r1 & 7)) * 16));
              if (row - lane + r1 < part.rows) {
                *reinterpret_cast<uint4*>(slot + (row - lane + r1) * D + col + 4 * piece) = x;
              }
            }
          }
          __syncwarp();
        }
        if (on && part.whole) {
          a.lse[at] = lsum == 0.f ? INFINITY : (top + log2f(lsum)) * kLn2;
        } else if (on) {
          slot[kRows * D + row] = top;
          slot[kRows * D + kRows + row] = lsum;
        }
      }
      if (merge) pair_barrier();  // group 1's sums were read
      first_part = false;
    } while (next_part());
  } else if (warp < 16) {
    // ---------------------------------------------------------------- conversion
    regs_dealloc<72>();
    constexpr int kPieces = D / 16, kStep = 128 / kPieces;  // kStep rows at a time
    const int is_v = warp >= 12;
    // Eight lanes that store together have two neighbouring rows and four pieces of one 128-byte
    // chunk: their swizzled places are in different banks.
    const int t = tid & 127;
    const int piece = (t & 3) + (D == 128 ? ((t >> 3) & 1) * 4 : 0);
    const int row0 = D == 128 ? ((t >> 2) & 1) + (t >> 4) * 2 : t >> 2;
    const uint32_t spot = sbase + (is_v ? L::kV16 : L::kK16) + (piece >> 2) * L::kChunkBytes + row0 * 128;
    const uint32_t lo = spot + (((piece & 3) * 2) ^ (row0 & 7)) * 16;
    const uint32_t hi = spot + (((piece & 3) * 2 + 1) ^ (row0 & 7)) * 16;
    const unsigned char* const base =
        (is_v ? c.v : c.k) + (row0 & 15) * (is_v ? c.vs[2] : c.ks[2]) + piece * 16;
    const int full = is_v ? L::kV16Full : L::kK16Full, empty = is_v ? L::kV16Empty : L::kK16Empty;
    unsigned n = 0;  // tiles stored
    bool ok = true;
    int i = 0, n_tiles = part.n_tiles;
    uint4 kv[kPieces];
    // This thread's pieces of tile i of the part, zeros where no key is.
    bool masked = false;  // V of a tile that not all rows see all of
    auto fetch = [&](unsigned at) {
      const int slot = at % kTables;
      const long long tokens = (part.tile0 + i + 1ll) * kKeys - (part.t.q.len - part.t.q.n) - 1;
      masked = is_v && a.causal && tokens * group > part.row0;
      ok = __all_sync(0xffffffffu,
                      wait_or_abort(bar(L::kTabFull + slot), (at / kTables) & 1, w, kStKFull));
      if (!ok) return;
      const long long* from = &tables[slot * kGroups + (row0 >> 4)].k_at + is_v;
      constexpr int kNext = sizeof(RunScale) / 8 * (kStep / 16);
      if (clean[slot]) {
#pragma unroll
        for (int x = 0; x < kPieces; ++x) kv[x] = ldg128(base + from[x * kNext]);
      } else {  // behind the last key a page holds anything, and 0 times that must be 0
        const RunScale* table = tables + slot * kGroups + (row0 >> 4);
        const int left = part.t.q.len - (part.tile0 + i) * kKeys;  // keys that are there
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
          kv[x] = make_uint4(0, 0, 0, 0);
          if (row0 + x * kStep < left && table[x * kStep / 16].page >= 0) {
            kv[x] = ldg128(base + from[x * kNext]);
          }
        }
      }
    };
    bool more = true;
    while (more && n_tiles == 0) {
      more = next_part();
      n_tiles = part.n_tiles;
    }
    if (more) fetch(0);
    while (more && ok) {
      const int st = n & 1;
      ok = n < 2 || wait_or_abort(bar(empty + st), ((n >> 1) & 1) ^ 1, w, kStKVEmpty);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (masked) {
        uint32_t nans = 0;
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
          const uint4 f = make_uint4(nan_bytes(kv[x].x), nan_bytes(kv[x].y), nan_bytes(kv[x].z),
                                     nan_bytes(kv[x].w));
          nans |= f.x | f.y | f.z | f.w;
          kv[x] = make_uint4(kv[x].x & ~f.x, kv[x].y & ~f.y, kv[x].z & ~f.z, kv[x].w & ~f.w);
        }
        if (nans != 0) atomicMax(last_nan, n + 1);
      }
#pragma unroll
      for (int x = 0; x < kPieces; ++x) {
        store_wide(lo + st * L::kTile16 + x * kStep * 128, hi + st * L::kTile16 + x * kStep * 128, kv[x]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(full + st));
      // The tile after this one, in this part or a later one.
      if (++i == n_tiles) {
        i = 0;
        do {
          more = next_part();
          n_tiles = part.n_tiles;
        } while (more && n_tiles == 0);
      }
      if (more) fetch(++n);
    }
  } else {
    regs_dealloc<64>();
    if (warp == 16) {
      // -------------------------------------------------------------- pages
      // Lane 8 b + x looks after 16 keys (run x) of tile b of four; pages are looked up four tiles
      // ahead, their scales a tile later.
      const int x = lane & 7;
      unsigned n = 0;  // tiles
      bool ok = true;
      do {
        const unsigned keys_end = min(part.t.q.len, (part.tile0 + part.n_tiles) * kKeys);
        const int head = part.p.head;
        // Unsigned: up to seven tiles ahead of a key that may be next to 2^31.
        auto key_at = [&](int i) {
          return static_cast<unsigned>(part.tile0 + i + (lane >> 3)) * kKeys + 16 * x;
        };
        auto page_at = [&](int i) {
          const unsigned key = key_at(i);
          return key < keys_end ? page_of(c, part.p.s, static_cast<int>(key >> c.page_shift)) : -1;
        };
        float sk = 0.f, sv = 1.f;
        auto read_scales = [&](int page) {
          if (page >= 0) {
            const long long at = static_cast<long long>(page) * c.Hkv + head;
            sk = __ldg(c.k_scale + at);
            sv = __ldg(c.v_scale + at);
          }
        };
        int next_page = part.n_tiles > 0 ? page_at(0) : -1;
        read_scales(next_page);
        RunScale sc = {0.f, 0.f, 0.f, -1, 0, 0};
        for (int i = 0; i < part.n_tiles && ok; ++i, ++n) {
          if ((i & 3) == 0) {
            const int slot = key_at(i) & ((1 << c.page_shift) - 1);
            sc.page = next_page;
            sc.mul = sk;
            value_scale(c, sv, &sc.add, &sc.inv);
            sc.k_at = next_page * c.ks[0] + head * c.ks[1] + slot * c.ks[2];
            sc.v_at = next_page * c.vs[0] + head * c.vs[1] + slot * c.vs[2];
            next_page = page_at(i + 4);
          }
          if ((i & 3) == 1) read_scales(next_page);
          const int slot = n % kTables;
          if (n >= kTables) {
            ok = __all_sync(0xffffffffu, wait_or_abort(bar(L::kTabEmpty + slot),
                                                       ((n / kTables) & 1) ^ 1, w, kStKVEmpty));
            if (!ok) break;
          }
          const bool mine = (lane >> 3) == (i & 3);
          if (mine) tables[slot * kGroups + x] = sc;
          const unsigned there = __ballot_sync(0xffffffffu, mine && sc.page >= 0);
          if (lane == 0) {
            clean[slot] = __popc(there) == kGroups &&
                          (part.tile0 + i + 1) * kKeys <= part.t.q.len;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(L::kTabFull + slot));
        }
      } while (ok && next_part());
    } else if (warp < 19) {
      // -------------------------------------------------------------- products, a warp for each group
      // The whole warp walks the schedule and one lane issues: with every operand the same in all
      // lanes the compiler keeps them in uniform registers, where the instructions want them.  Two
      // warps, since the time from one product's issue to the next wait (about 500 cycles) is as long
      // as the products.
      constexpr uint32_t kIdescS = idesc_mma(0, 128, kKeys / 2, false);
      constexpr uint32_t kIdescPV = idesc_mma(0, 128, D, true);
      constexpr uint32_t kHalfBytes = (kKeys / 2) * 128;  // 64 keys of a 128-byte chunk
      const int g = __shfl_sync(0xffffffffu, warp - 17, 0);
      const uint32_t base = __shfl_sync(0xffffffffu, sbase, 0);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t s_tm = tm + L::kColS + g * 128, o_tm = tm + L::kColO + g * 128;
      const uint64_t q_desc = sdesc_sw128(base + L::kQ, 16, 1024);
      const uint64_t k_desc = sdesc_sw128(base + L::kK16, 16, 1024);
      const uint64_t v_desc = sdesc_sw128(base + L::kV16, L::kChunkBytes, 1024);
      auto all = [](bool x) { return __all_sync(0xffffffffu, x); };
      unsigned tiles_done = 0, my_tiles = 0, parts_done = 0, q1_done = 0;
      bool ok = true;
      do {
        // With more than 128 rows both groups have every tile, otherwise this one has tiles g, g + 2,
        // ... and stands in for the other where both have to give a buffer back.
        const bool pair = __shfl_sync(0xffffffffu, static_cast<int>(part.pair), 0);
        const int n_tiles = __shfl_sync(0xffffffffu, part.n_tiles, 0);
        const int step = pair ? 2 : 1;
        const uint64_t qd = q_desc + (pair ? 0 : (g * L::kTile16) >> 4);
        auto issue_s = [&](int i, int h) -> bool {
          if (i >= n_tiles) return true;
          const unsigned tile = tiles_done + i;
          const int st = tile & 1;
          if (h == 0) {
            if (!all(wait_or_abort(bar(L::kK16Full + st), (tile >> 1) & 1, w, kStKFull))) return false;
            tc_fence_after();
          }
          const uint64_t kd = k_desc + ((st * L::kTile16 + h * kHalfBytes) >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = (kk / 4) * L::kChunkBytes + (kk % 4) * 32;
              umma_ss(s_tm + h * 64, qd + (off >> 4), kd + (off >> 4), kIdescS, kk > 0 ? 1u : 0u);
            }
            umma_commit(bar(L::kSFull + 2 * g + h));
            if (h == 1) {
              umma_commit(bar(L::kK16Empty + st));
              if (pair) umma_commit(bar(L::kK16Empty + st));
            }
          }
          __syncwarp();
          return true;
        };
        auto issue_pv = [&](int i, int h) -> bool {
          const unsigned tile = tiles_done + i;
          const int st = tile & 1;
          if (!all(wait_or_abort(bar(L::kPFull + 2 * g + h), my_tiles & 1, w, kStPFull))) return false;
          if (h == 0) {
            if (!all(wait_or_abort(bar(L::kV16Full + st), (tile >> 1) & 1, w, kStVFull))) return false;
          }
          tc_fence_after();
          const uint64_t vd = v_desc + ((st * L::kTile16 + h * kHalfBytes) >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kKeys / 32; ++kk) {
              umma_ts(o_tm, s_tm + h * 64 + 8 * kk, vd + ((kk * 2048) >> 4), kIdescPV,
                      (i >= step || h > 0 || kk > 0) ? 1u : 0u);
            }
            umma_commit(bar(L::kODone + g));
            if (h == 1) {
              if (i + step >= n_tiles) umma_commit(bar(L::kOFull + g));
              umma_commit(bar(L::kV16Empty + st));
              // Both the weights and V's buffer of this tile are done with its table.
              mbar_arrive(bar(L::kTabEmpty + tile % kTables));
              if (pair) {
                umma_commit(bar(L::kV16Empty + st));
                mbar_arrive(bar(L::kTabEmpty + tile % kTables));
              }
            }
          }
          __syncwarp();
          if (h == 1) ++my_tiles;
          return true;
        };
        const int first = pair ? g : 0;
        if (n_tiles > 0) {
          // Group 0's Q even where this group reads its own: the barrier's phases count parts.
          ok = all(wait_or_abort(bar(L::kQFull), parts_done & 1, w, kStQFull));
          ++parts_done;
          if (g == 1 && !pair) {
            ok = ok && all(wait_or_abort(bar(L::kQFull + 1), q1_done & 1, w, kStQFull));
            ++q1_done;
          }
          tc_fence_after();
        }
        ok = ok && issue_s(first, 0) && issue_s(first, 1);
        // S of the next tile follows the PV that read P from its columns: products that one thread
        // issues execute in order.
        for (int i = first; i < n_tiles && ok; i += step) {
#pragma unroll
          for (int h = 0; h < 2; ++h) ok = ok && issue_pv(i, h) && issue_s(i + step, h);
        }
        tiles_done += n_tiles;
      } while (ok && next_part());
      if (elect_one()) umma_commit(bar(L::kDrain));
      __syncwarp();
      wait_out(bar(L::kDrain), 0, w);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 17) tmem_dealloc(tmem, L::kCols);
}

// Merges the parts of a tile that several CTAs share.  Block i looks after the tile that CTA i's range
// begins inside of, if no earlier CTA's does too; a warp for each row, kMergeBlocks blocks for a tile (one:
// 26 us where CTAs share 147 tiles of 256 rows).
constexpr int kMergeBlocks = 4, kMergeThreads = 256;
template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) fa_cache_tile_merge_kernel(
    const __grid_constant__ CacheAttnArgs a, const float* partials) {
  using L = Layout<D>;
  constexpr int kPer = D / 32, kWarps = kMergeThreads / 32, kBatch = 4;
  __shared__ Finder<kMergeThreads> finder;
  const CacheView& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = a.H / c.Hkv;
  const int me = blockIdx.x;
  long long per;
  const long long total = finder.find(c, group, a.causal, me, &per);
  const long long begin = me * per;
  const Place p = finder.at;
  wait_for_parts();
  if (me == 0 || begin >= total || p.tile == 0 || p.tile > per) return;
  const SeqTiles t = tiles_of(finder.q, group, a.causal);
  const long long first = begin - p.tile, end = first + t.of(p.j, group);
  const int last = static_cast<int>((end - 1) / per);  // the last CTA with a part
  const int row0 = p.j * kRows, rows = min(kRows, t.rows - row0);
  for (int row = blockIdx.y * kWarps + warp; row < rows; row += gridDim.y * kWarps) {
    float top = -INFINITY, lsum = 0.f, acc[kPer] = {};
    for (int i0 = me - 1; i0 <= last; i0 += kBatch) {
      float pm[kBatch], pl[kBatch], v[kBatch][kPer];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        pm[b] = -INFINITY;
        pl[b] = 0.f;
        if (i0 + b <= last) {
          const int slot = (i0 + b) * per >= first ? 0 : 1;
          const float* part = partials + (2ll * (i0 + b) + slot) * L::kPartial;
          pm[b] = part[kRows * D + row];
          pl[b] = part[kRows * D + kRows + row];
#pragma unroll
          for (int k = 0; k < kPer; ++k) v[b][k] = part[row * D + lane * kPer + k];
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (pm[b] == -INFINITY && pl[b] == 0.f) continue;
        const float to = fmaxf(top, pm[b]);
        const float f0 = top == -INFINITY ? 1.f : ex2_approx(top - to);
        const float f1 = pm[b] == -INFINITY ? 1.f : ex2_approx(pm[b] - to);
        top = to;
        lsum = lsum * f0 + pl[b] * f1;
#pragma unroll
        for (int k = 0; k < kPer; ++k) acc[k] = acc[k] * f0 + v[b][k] * f1;
      }
    }
    const int token = (row0 + row) / group;
    const long long at = static_cast<long long>(t.q.t0 + token) * a.H + p.head * group +
                         (row0 + row - token * group);
    const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
    uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<T*>(a.o) + at * D + lane * kPer);
#pragma unroll
    for (int k = 0; k < kPer; k += 2) o[k / 2] = from_float2<T>(acc[k] * inv, acc[k + 1] * inv);
    if (lane == 0) a.lse[at] = lsum == 0.f ? INFINITY : (top + log2f(lsum)) * kLn2;
  }
}

template <typename T, int D>
cudaError_t launch_t(const CacheAttnArgs& a, cudaStream_t stream) {
  using L = Layout<D>;
  const CacheView& c = a.c;
  const int group = a.H / c.Hkv;
  // No more CTAs than units that the table could hold.
  const long long room = static_cast<long long>(c.max_pages) << c.page_shift;
  const long long units = std::max(1ll, (room + kKeys - 1) / kKeys);
  const long long tiles = (static_cast<long long>(c.T) * group / kRows + c.n_seqs) * c.Hkv;
  const long long want = tiles > (1ll << 40) / units ? (1ll << 40) : tiles * units;
  const unsigned ctas =
      static_cast<unsigned>(std::max(1ll, std::min<long long>(multiprocessors(), want)));
  float* partials = static_cast<float*>(a.workspace);
  cudaError_t e =
      cudaFuncSetAttribute(fa_cache_tile_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           L::kBytes);
  if (e != cudaSuccess) return e;
  fa_cache_tile_kernel<T, D><<<ctas, kThreads, L::kBytes, stream>>>(a, partials);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if (units == 1) return cudaSuccess;  // no tile has two units: none has more than its sequence's keys
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, kMergeBlocks);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fa_cache_tile_merge_kernel<T, D>, a,
                            static_cast<const float*>(partials));
}

}  // namespace

size_t cache_tile_workspace(int D, int sms) {
  const size_t floats = D == 64 ? Layout<64>::kPartial : Layout<128>::kPartial;
  return 2 * sizeof(float) * static_cast<size_t>(sms) * floats;
}

cudaError_t launch_cache_tile(const CacheAttnArgs& a, cudaStream_t stream) {
  if (a.dtype == FA_DTYPE_F16) {
    return a.D == 64 ? launch_t<__half, 64>(a, stream) : launch_t<__half, 128>(a, stream);
  }
  return a.D == 64 ? launch_t<__nv_bfloat16, 64>(a, stream)
                   : launch_t<__nv_bfloat16, 128>(a, stream);
}

}  // namespace fa_sm100
