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
// queries), and costs one term for a run of 16 keys, since a run never leaves its page.  In return P is
// rounded relative to the row's largest P sv: 11 bits down to 2^-14 of it, and below 2^-25 of it a key is
// in the denominator alone.  The denominator is a sum in 32 bits; P has to stay above 2^-126 for it, so
// value scales have a range (value_scale) and those of one sequence lie within 2^96 of each other.
//
// bf16 queries enter the products as fp16 after division by a power of two for each row: 8
// significant bits fit in fp16's 11, so this is exact but for values 2^-23 below the row's largest.
//
// A query row is (token, head of the group), so a kv head's keys are read once for all of its heads.
// Up to 32 rows of a sequence go through mma.sync with the keys as M and 8 rows as N: tcgen05's 128
// rows would be mostly padding, and the bytes of the cache, not the products, bound these calls.  Each
// warp takes runs of 16 keys from a ring that TMA fills, with its own maximum and sum; nothing in the
// loop waits for another warp.  All sequences' units of 64 keys are numbered and split evenly over the
// CTAs (lengths live on the device, so a captured call follows them); tiles that several CTAs share
// leave fp32 partials, which a second kernel, launched while the first runs, merges.
//
// What bounds it: 64 sequences of 97 to 8191 keys of 8 heads of 128, one token of 32 heads each, 554 MB,
// take 111 us (84 at the measured copy rate), one of 131071 keys, 269 MB, 63 us (41): 5.9 TB/s between the
// two and some 18 us that do not depend on the length (the table's and the first page's latency, the merge);
// the kernel alone reads 5.2 to 5.4 TB/s.  5 tokens of 32 heads, 20 rows, take 71 us for 153 MB: the
// products' instructions and the softmax of 24 rows.  777 keys take 12.6 us, two kernels of some 7 us that
// are chains of latencies.  One sequence's tables were looked up by each run before (142 us for the first of
// these), rows as M (171 us).
#include <algorithm>
#include <cmath>

#include "fa_cache_common.cuh"
#include "sm100_ptx.cuh"

namespace fa_sm100 {
namespace {

constexpr int kRun = 16;    // keys that a warp takes at a time; never more than a page
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = kRun * kWarps;  // keys of one unit of work
constexpr float kLazy = 8.0f;         // the running maximum follows once it is off by 2^8
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;

// A CTA's tile has 8 NT query rows (token, head of the group).
template <int D, int NT>
struct Layout {
  static constexpr int kRows = 8 * NT;
  static constexpr int kStages = D == 128 && NT == 1 ? 3 : 4;  // runs in flight for each warp
  // CTAs on a multiprocessor: as many as the accumulators' registers leave room for.
  static constexpr int kPerSm = NT > 2 ? 2 : D == 128 ? (NT == 1 ? 4 : 3) : (NT == 1 ? 5 : 4);
  static constexpr int kHalf = kRun * D;  // K or V bytes of a run
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kMerge = kWarps * kRows * D * 4;  // reuses the ring
  static constexpr int kMain = kRing > kMerge ? kRing : kMerge;
  static constexpr int kScale = kWarps * 64 * 16;
  static constexpr int kBars = kWarps * kStages * 8;
  static constexpr int kBytes = kMain + kScale + kBars + 1024;  // the ring starts on 1024 bytes
  // A partial result: kRows x D sums, then (m, l) of each row.
  static constexpr int kPartial = kRows * D + 2 * kRows;
};

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

template <int ROWS>
__device__ __forceinline__ SeqWork work_of(const SeqInfo& q, int group) {
  SeqWork w;
  w.q = q;
  w.row_tiles = (w.q.n * group + ROWS - 1) / ROWS;
  w.tiles = max(1, (w.q.len + kTile - 1) / kTile);
  return w;
}

template <int ROWS>
__device__ __forceinline__ SeqWork seq_work(const CacheView& c, int s, int group) {
  return work_of<ROWS>(seq_info(c, s), group);
}

// Units are numbered sequence by sequence; CTA i of ceil(total / per) takes [i per, (i + 1) per).
// Whole multiples keep the longest range as short as an even split would, with fewer CTAs that share
// a tuple, and make the inverse one division.
__device__ __forceinline__ long long units_per_cta(long long total) {
  return (total + gridDim.x - 1) / gridDim.x;
}

struct Place {
  int s;            // sequence of the unit
  SeqInfo q;
  long long first;  // its first unit
};

// Every CTA adds up the units of all sequences and finds the one that its own range begins in.  The
// lengths live on the device, so that a captured call follows them; THREADS sequences at a time.
template <int THREADS, int ROWS>
struct Finder {
  long long warp[THREADS / 32];
  long long first;  // unit that the range begins with
  Place at;

  // Sums x over the block up to and including this thread; *sum is the block's.
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

  // The total of units.  With at most THREADS sequences `mine` and `incl` are this thread's for find.
  __device__ long long total(const CacheView& c, int group, SeqWork* w, long long* incl) {
    if (threadIdx.x == 0) at = Place{0, SeqInfo{0, 0, 0}, 0};
    long long run = 0, sum;
    for (int base = 0; base < c.n_seqs; base += THREADS) {
      const int s = base + threadIdx.x;
      *w = s < c.n_seqs ? seq_work<ROWS>(c, s, group) : SeqWork{SeqInfo{0, 0, 0}, 0, 1};
      *incl = scan(w->units(c.Hkv), &sum);
      run += sum;
    }
    return run;
  }

  __device__ void find(const CacheView& c, int group, SeqWork w, long long incl, long long unit) {
    long long run = 0, sum;
    for (int base = 0; base < c.n_seqs; base += THREADS) {
      const int s = base + threadIdx.x;
      if (c.n_seqs > THREADS) {
        w = s < c.n_seqs ? seq_work<ROWS>(c, s, group) : SeqWork{SeqInfo{0, 0, 0}, 0, 1};
        incl = run + scan(w.units(c.Hkv), &sum);
        run += sum;
      }
      const long long mine = w.units(c.Hkv);
      if (unit < incl && unit >= incl - mine) at = Place{s, w.q, incl - mine};
    }
    __syncthreads();
  }
};

// Bounded wait for a phase of this warp's copies; false when the time limit ran out (reported).
__device__ __forceinline__ bool wait_copy(uint32_t bar, uint32_t parity, const CacheView& c,
                                          unsigned long long timeout_ns) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > timeout_ns) {
      atomicOr(c.status, kStKFull);
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

// An 8 x 8 block of 16-bit values, two of a row to a lane, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t u) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(u));
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
  int page;  // -1: the run's keys count as absent
};

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

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, (Layout<D, NT>::kPerSm)) fa_cache_decode_kernel(
    const __grid_constant__ CacheAttnArgs a, const __grid_constant__ PageMaps maps,
    float* partials) {
  using L = Layout<D, NT>;
  constexpr int kRows = L::kRows;
  constexpr int kSteps = D / 16;   // products of 16 along D
  constexpr int kPieces = D / 16;  // 16-byte pieces of a K or V row
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ Finder<kThreads, kRows> finder;
  __shared__ float merge_m[kWarps][kRows], merge_l[kWarps][kRows];

  const CacheView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = lane >> 2, cq = lane & 3;  // row and column group of the fragments
  const int group = a.H / c.Hkv;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  zero_stray_rows<T, D, kThreads>(a);

  SeqWork w;
  long long incl;
  const long long total = finder.total(c, group, &w, &incl);
  const long long per = units_per_cta(total);
  const long long u_begin = blockIdx.x * per, u_end = min(total, u_begin + per);
  if (u_begin >= u_end) return;
  finder.find(c, group, w, incl, u_begin);
  int s = finder.at.s;
  long long seq_first = finder.at.first;
  w = work_of<kRows>(finder.at.q, group);

  const uint32_t ring = smem_u32(smem) + warp * L::kStages * L::kStage;
  RunScale* table = reinterpret_cast<RunScale*>(smem + L::kMain) + warp * 64;
  const uint32_t bars = smem_u32(smem) + L::kMain + L::kScale + warp * L::kStages * 8;
  const int page_mask = (1 << c.page_shift) - 1;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < L::kStages; ++i) mbar_init(bars + 8 * i, 1);
    fence_mbar_init();
  }
  __syncwarp();
  unsigned sent = 0, taken = 0;  // runs that this warp has issued and used, over all parts
  bool alive = true;             // false once a wait ran out: nothing more is issued or used

  for (long long u = u_begin; u < u_end;) {
    while (u >= seq_first + w.units(c.Hkv)) {  // on to the sequence of unit u
      if (s + 1 >= c.n_seqs) return;
      seq_first += w.units(c.Hkv);
      w = seq_work<kRows>(c, ++s, group);
    }
    const long long tuple = (u - seq_first) / w.tiles;
    const int tile0 = static_cast<int>(u - seq_first - tuple * w.tiles);
    const int tile1 = static_cast<int>(min(static_cast<long long>(w.tiles), tile0 + (u_end - u)));
    const int head = static_cast<int>(tuple / w.row_tiles);
    const int row0 = static_cast<int>(tuple - static_cast<long long>(head) * w.row_tiles) * kRows;
    const int rows = min(kRows, w.q.n * group - row0);

    // Keys that the tile's last row sees, and those that all of its rows see.
    const int last_token = (row0 + rows - 1) / group, first_token = row0 / group;
    const int seen = a.causal ? max(0, w.q.len - w.q.n + last_token + 1) : w.q.len;
    const int all_see = a.causal ? max(0, w.q.len - w.q.n + first_token + 1) : w.q.len;

    // Runs of this warp: keys [first_key + i * kTile, + kRun), i < n_runs.
    const int first_key = tile0 * kTile + warp * kRun;
    const int stop = min(seen, tile1 * kTile);
    const int n_runs = first_key < stop ? (stop - first_key + kTile - 1) / kTile : 0;

    // Pages and scales of 32 runs at a time, a lane each, a batch ahead of their use: the page when
    // run 4 of the batch before is issued, its scales 8 runs later, both into the table 8 runs later.
    static_assert(L::kStages <= 4, "the first runs are issued without this schedule");
    auto page_at = [&](int i) {
      return i < n_runs ? page_of(c, s, (first_key + i * kTile) >> c.page_shift) : -1;
    };
    int page = page_at(lane);
    float sk = 0.f, sv = 1.f;
    auto read_scales = [&]() {
      if (page >= 0) {
        const long long at = static_cast<long long>(page) * c.Hkv + head;
        sk = __ldg(c.k_scale + at);
        sv = __ldg(c.v_scale + at);
      }
    };
    auto write_table = [&](int i) {
      RunScale sc;
      sc.mul = sk;
      value_scale(c, sv, &sc.add, &sc.inv);
      sc.page = page;
      table[i & 63] = sc;
      __syncwarp();
    };
    auto send = [&](int i, int pg) {  // by one lane: run i's copies into the next stage
      const int stage = sent % L::kStages;
      const uint32_t bar = bars + 8 * stage, dst = ring + stage * L::kStage;
      if (pg >= 0) {
        const int slot = (first_key + i * kTile) & page_mask;
        mbar_arrive_expect_tx(bar, L::kStage);
        load_page(dst, &maps.k, maps.k_pos, slot, head, pg, bar);
        load_page(dst + L::kHalf, &maps.v, maps.v_pos, slot, head, pg, bar);
      } else {
        mbar_arrive(bar);
      }
    };
    int issued = 0;
#pragma unroll
    for (int i = 0; i < L::kStages - 1; ++i, ++issued) {  // before the scales are known
      const int pg = __shfl_sync(0xffffffffu, page, i);
      if (i < n_runs && alive) {
        if (lane == 0) send(i, pg);
        ++sent;
      }
    }
    read_scales();
    auto issue = [&]() {
      const int i = issued++;
      if (i >= n_runs) return;
      const int step = i & 31;
      if (step == 4) page = page_at(i + 28 + lane);
      if (step == 12) read_scales();
      if (step == 20) write_table(i + 12 + lane);
      if (lane == 0) send(i, table[i & 63].page);
      ++sent;
    };

    // Query row r of each 8: the B fragments.  Columns of step t are 4 neighbours of a row, so that
    // a K word is the two halves of an A fragment.
    uint32_t qf[NT][kSteps][2];
    int limit[NT][2];      // visible keys of the rows 2cq, 2cq + 1 of each 8 (C fragments)
    float row_mul[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int row = row0 + 8 * x + r;
      const bool on = 8 * x + r < rows;
      const int token = on ? row / group : 0;
      const int h = head * group + (on ? row - token * group : 0);
      int lim = on ? (a.causal ? max(0, w.q.len - w.q.n + token + 1) : w.q.len) : 0;
      const T* src = static_cast<const T*>(a.q) + (w.q.t0 + token) * a.sq[0] + h * a.sq[1];
      uint32_t(&raw)[kSteps][2] = qf[x];
#pragma unroll
      for (int p = 0; p < kSteps / 4; ++p) {
        const uint4* at = reinterpret_cast<const uint4*>(src + 16 * k_piece<D>(cq, p));
        const uint4 v0 = on ? __ldg(at) : make_uint4(0, 0, 0, 0);
        const uint4 v1 = on ? __ldg(at + 1) : make_uint4(0, 0, 0, 0);
        const uint32_t f[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[4 * p + i / 2][i & 1] = f[i];
      }
      float mul = a.scale * kLog2e;
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
                          ? min(119, max(-118, static_cast<int>(__float_as_uint(big) >> 23) - 127 - 8))
                          : 0;
        const float div = __int_as_float((127 - e) << 23);
        mul *= __int_as_float((127 + e) << 23);
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
      for (int e = 0; e < 2; ++e) {
        limit[x][e] = __shfl_sync(0xffffffffu, lim, (2 * cq + e) * 4);
        row_mul[x][e] = __shfl_sync(0xffffffffu, mul, (2 * cq + e) * 4);
      }
    }
    write_table(lane);

    // Sums transposed: columns (D / 8) r + 2 j + (e >> 1), row 2cq + (e & 1) of each 8.
    float acc[NT][D / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[x][j][e] = 0.f;
      }
      m[x][0] = m[x][1] = -INFINITY;
      l[x][0] = l[x][1] = 0.f;
    }

    uint32_t nans = 0;  // V's NaN that were taken out (nan_columns)
    for (int i = 0; i < n_runs; ++i) {
      const int stage = taken % L::kStages;
      if (alive) alive = wait_copy(bars + 8 * stage, (taken / L::kStages) & 1, c, a.timeout_ns);
      alive = __all_sync(0xffffffffu, alive);
      if (!alive) break;
      ++taken;
      issue();  // into the stage that every lane left before the vote
      const uint32_t kb = ring + stage * L::kStage;
      const uint32_t vb = kb + L::kHalf;
      const RunScale sc = table[i & 63];

      // Scores, transposed: keys r, r + 8 by rows 2cq, 2cq + 1.  Even and odd steps apart, for
      // shorter chains of products.
      float sacc[NT][2][4] = {};
#pragma unroll
      for (int p = 0; p < kPieces / 4; ++p) {
        const int piece = k_piece<D>(cq, p);
        const uint32_t at =
            kb + r * D + (D == 128 ? piece ^ r : piece ^ ((r >> 1) & 3)) * 16;
        const uint4 lo = lds128(at), hi = lds128(at + 8 * D);
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t kf[4] = {e4m3_lo(wl[t]), e4m3_lo(wh[t]), e4m3_hi(wl[t]), e4m3_hi(wh[t])};
#pragma unroll
          for (int x = 0; x < NT; ++x) mma_f16(sacc[x][t & 1], kf, qf[x][4 * p + t][0], qf[x][4 * p + t][1]);
        }
      }

      float t[NT][4];
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        const float mul[2] = {sc.mul * row_mul[x][0], sc.mul * row_mul[x][1]};
#pragma unroll
        for (int e = 0; e < 4; ++e) t[x][e] = fmaf(sacc[x][0][e] + sacc[x][1][e], mul[e & 1], sc.add);
      }
      const int key0 = first_key + i * kTile;
      const bool masked = key0 + kRun > all_see || sc.page < 0;
      if (masked) {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (sc.page < 0 || key0 + r + 8 * (e >> 1) >= limit[x][e & 1]) t[x][e] = -INFINITY;
          }
        }
      }
      bool moved = false;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
#pragma unroll
        for (int e = 0; e < 2; ++e) moved |= fmaxf(t[x][e], t[x][e + 2]) > m[x][e] + kLazy;
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float big = fmaxf(t[x][e], t[x][e + 2]);
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 4));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 8));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 16));
            const float to = fmaxf(m[x][e], big);
            const float f = to == m[x][e] ? 1.f : ex2_approx(m[x][e] - to);
            m[x][e] = to;
            l[x][e] *= f;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              acc[x][j][e] *= f;
              acc[x][j][e + 2] *= f;
            }
          }
        }
      }
      uint32_t pf[NT][2];  // P's B fragments: the 8 x 8 blocks of P transposed
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = ex2_approx(t[x][e] - (m[x][e & 1] == -INFINITY ? 0.f : m[x][e & 1]));
        }
        l[x][0] = fmaf(p[0] + p[2], sc.inv, l[x][0]);
        l[x][1] = fmaf(p[1] + p[3], sc.inv, l[x][1]);
        pf[x][0] = transpose8(from_float2<__half>(p[0], p[1]));
        pf[x][1] = transpose8(from_float2<__half>(p[2], p[3]));
      }

      // V, transposed: this lane's keys 2cq, 2cq + 1, 2cq + 8, 2cq + 9 and columns (D / 8) r + ...
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
      if (masked) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // a page's tail holds anything
          const bool there = sc.page >= 0 && key0 + 2 * cq + (k & 1) + 8 * (k >> 1) < w.q.len;
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const uint32_t v = there ? vw[k][j] : 0, n = nan_bytes(v);
            vw[k][j] = v & ~n;
            nans |= n;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {  // columns 4j .. 4j + 3 of the lane's
        const uint32_t a0 = __byte_perm(vw[0][j], vw[1][j], 0x5140);
        const uint32_t a1 = __byte_perm(vw[0][j], vw[1][j], 0x7362);
        const uint32_t b0 = __byte_perm(vw[2][j], vw[3][j], 0x5140);
        const uint32_t b1 = __byte_perm(vw[2][j], vw[3][j], 0x7362);
        const uint32_t v0[4] = {e4m3_lo(a0), e4m3_hi(a0), e4m3_lo(b0), e4m3_hi(b0)};
        const uint32_t v1[4] = {e4m3_lo(a1), e4m3_hi(a1), e4m3_lo(b1), e4m3_hi(b1)};
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          mma_f16(acc[x][2 * j], v0, pf[x][0], pf[x][1]);
          mma_f16(acc[x][2 * j + 1], v1, pf[x][0], pf[x][1]);
        }
      }
    }
    // Copies in flight when a wait ran out still write to this block's memory.
    while (taken != sent) {
      wait_copy(bars + 8 * (taken % L::kStages), (taken / L::kStages) & 1, c, max(a.timeout_ns, kMinDrainNs));
      ++taken;
    }

    // Merge the warps' sums: each scales its own to the block's maximum, then the block adds.
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o *= 2) l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], o);
        if (r == 0) {
          merge_m[warp][8 * x + 2 * cq + e] = m[x][e];
          merge_l[warp][8 * x + 2 * cq + e] = l[x][e];
        }
      }
    }
    const bool spoiled = __syncthreads_or(nans != 0);  // and no warp reads its ring any more
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 8 * x + 2 * cq + e;
        float top = merge_m[0][row];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) top = fmaxf(top, merge_m[i][row]);
        const float f = m[x][e] == -INFINITY ? (l[x][e] == l[x][e] ? 0.f : l[x][e])
                                             : ex2_approx(m[x][e] - top);
        float* at = sums + (warp * kRows + row) * D + r * (D / 8);
#pragma unroll
        for (int j = 0; j < D / 16; j += 2) {
          *reinterpret_cast<float4*>(at + 2 * j) =
              make_float4(acc[x][j][e] * f, acc[x][j][e + 2] * f, acc[x][j + 1][e] * f,
                          acc[x][j + 1][e + 2] * f);
        }
      }
    }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == w.tiles;
#pragma unroll 1
    for (int e = tid; e < rows * (D / 8); e += kThreads) {  // 8 columns of a row at a time
      const int row = e / (D / 8), col = (e % (D / 8)) * 8;
      float top = merge_m[0][row], lsum = 0.f;
#pragma unroll
      for (int i = 1; i < kWarps; ++i) top = fmaxf(top, merge_m[i][row]);
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float wm = merge_m[i][row], wl = merge_l[i][row];
        lsum += wm == -INFINITY ? (wl == wl ? 0.f : wl) : wl * ex2_approx(wm - top);
      }
      float4 out[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        out[k] = *reinterpret_cast<const float4*>(sums + row * D + col + 4 * k);
#pragma unroll
        for (int i = 1; i < kWarps; ++i) {
          const float4 x =
              *reinterpret_cast<const float4*>(sums + (i * kRows + row) * D + col + 4 * k);
          out[k].x += x.x, out[k].y += x.y, out[k].z += x.z, out[k].w += x.w;
        }
      }
      const int token = (row0 + row) / group;
      if (spoiled) {
        const int see = a.causal ? max(0, w.q.len - w.q.n + token + 1) : w.q.len;
        const uint32_t bits = nan_columns<8>(c, s, head, max(tile0 * kTile, all_see & ~(kRun - 1)),
                                             min(see, tile1 * kTile), col);
        const float nan = __int_as_float(0x7fffffff);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (bits >> (4 * k) & 1) out[k].x = nan;
          if (bits >> (4 * k) & 2) out[k].y = nan;
          if (bits >> (4 * k) & 4) out[k].z = nan;
          if (bits >> (4 * k) & 8) out[k].w = nan;
        }
      }
      if (whole) {
        const long long at = static_cast<long long>(w.q.t0 + token) * a.H + head * group +
                             (row0 + row - token * group);
        const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
        uint4 v;
        v.x = from_float2<T>(out[0].x * inv, out[0].y * inv);
        v.y = from_float2<T>(out[0].z * inv, out[0].w * inv);
        v.z = from_float2<T>(out[1].x * inv, out[1].y * inv);
        v.w = from_float2<T>(out[1].z * inv, out[1].w * inv);
        *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + at * D + col) = v;
        if (col == 0) a.lse[at] = lsum == 0.f ? INFINITY : (top + log2f(lsum)) * kLn2;
      } else {
        float* part = partials + (2ll * blockIdx.x + (u == u_begin ? 0 : 1)) * L::kPartial;
        *reinterpret_cast<float4*>(part + row * D + col) = out[0];
        *reinterpret_cast<float4*>(part + row * D + col + 4) = out[1];
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

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * kCombineWarps) fa_cache_combine_kernel(
    const __grid_constant__ CacheAttnArgs a, const float* partials) {
  using L = Layout<D, NT>;
  constexpr int kRows = L::kRows;
  constexpr int kPer = D / 32;
  __shared__ Finder<32 * kCombineWarps, kRows> finder;
  __shared__ float sums[kCombineWarps][D];
  __shared__ float tops[kCombineWarps], lsums[kCombineWarps];
  const CacheView& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = a.H / c.Hkv;
  const int me = blockIdx.x;
  SeqWork w;
  long long incl;
  const long long total = finder.total(c, group, &w, &incl);
  const long long per = units_per_cta(total), begin = me * per;
  if (me == 0 || begin >= total) {
    wait_for_parts();
    return;
  }
  finder.find(c, group, w, incl, begin);
  const long long seq_first = finder.at.first;
  w = work_of<kRows>(finder.at.q, group);
  const long long tuple = (begin - seq_first) / w.tiles;
  const long long first = seq_first + tuple * w.tiles, end = first + w.tiles;
  wait_for_parts();
  if (first == begin || begin - per > first) return;
  const int head = static_cast<int>(tuple / w.row_tiles);
  const int row0 = static_cast<int>(tuple - static_cast<long long>(head) * w.row_tiles) * kRows;
  const int rows = min(kRows, w.q.n * group - row0);

  int split = 1;  // rows side by side; the warps of a row share its parts
  while (split < rows && split < kCombineWarps) split *= 2;
  const int share = warp / split, shares = kCombineWarps / split;
  const int last = static_cast<int>((end - 1) / per);  // the last CTA with a part
  for (int row = warp % split; row - warp % split < rows; row += split) {
    float top = -INFINITY, lsum = 0.f, acc[kPer] = {};
    if (row < rows) {
      constexpr int kBatch = 4;  // parts in flight
      for (int i0 = me - 1 + share; i0 <= last; i0 += kBatch * shares) {
        float pm[kBatch], pl[kBatch], v[kBatch][kPer];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int i = i0 + b * shares;
          pm[b] = -INFINITY;
          pl[b] = 0.f;
          if (i <= last) {
            // Its first part, unless it is the one that this tuple starts inside of.
            const int slot = i * per >= first ? 0 : 1;
            const float* part = partials + (2ll * i + slot) * L::kPartial;
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
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) sums[warp][lane * kPer + k] = acc[k];
    if (lane == 0) {
      tops[warp] = top;
      lsums[warp] = lsum;
    }
    __syncthreads();
    if (share == 0 && row < rows) {
      for (int i = 1; i < shares; ++i) {
        const int other = warp + i * split;
        const float pm = tops[other], pl = lsums[other];
        if (pm == -INFINITY && pl == 0.f) continue;
        const float to = fmaxf(top, pm);
        const float f0 = top == -INFINITY ? 1.f : ex2_approx(top - to);
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
    __syncthreads();  // the next rows' sums take the place of these
  }
}

template <typename T, int D, int NT>
cudaError_t launch_t(const CacheAttnArgs& a, cudaStream_t stream) {
  using L = Layout<D, NT>;
  const CacheView& c = a.c;
  const int group = a.H / c.Hkv;
  // No more CTAs than units that the table could hold.
  const long long room = static_cast<long long>(c.max_pages) << c.page_shift;
  const long long tiles = std::max(1ll, (room + kTile - 1) / kTile);
  const long long tuples =
      (static_cast<long long>(c.T) * group / L::kRows + c.n_seqs) * c.Hkv;
  const long long want = std::min<long long>(static_cast<long long>(L::kPerSm) * multiprocessors(),
                                             tuples > (1ll << 40) / tiles ? (1ll << 40) : tuples * tiles);
  const unsigned ctas = static_cast<unsigned>(std::max(1ll, want));
  float* partials = static_cast<float*>(a.workspace);
  PageMaps maps;
  cudaError_t e = make_page_maps(&maps, c, D, kRun);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(fa_cache_decode_kernel<T, D, NT>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  if (e != cudaSuccess) return e;
  fa_cache_decode_kernel<T, D, NT><<<ctas, kThreads, L::kBytes, stream>>>(a, maps, partials);
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
  return cudaLaunchKernelEx(&cfg, fa_cache_combine_kernel<T, D, NT>, a,
                            static_cast<const float*>(partials));
}

// Query rows of a tile in eights, by a sequence's mean; 0: the kernel on tcgen05 (fa_cache_tile.cu).
// 32 sequences of 500 to 4003 keys, rows: this kernel / the other, us.  32 + 8 heads of 128: 16: 58 / 107,
// 32: 93 / 110, 36: 157 / 112, 64: 172 / 113; 16 + 4 heads of 64: 32: 37 / 52, 36: 52 / 52, 64: 55 / 53,
// 128: 99 / 58.  Those batches are even.  For a skewed one the mean is a poor rule: 63 single tokens over
// 500 to 4003 keys and a chunk of 200 (500) over 4000 take 179 (273) us in one call, 137 (151) in two.
int row_eights(int H, int Hkv, int T, int n_seqs) {
  const long long rows = static_cast<long long>(T) * (H / Hkv);
  return rows > 32ll * n_seqs ? 0 : static_cast<int>(std::max(1ll, (rows + 8ll * n_seqs - 1) / (8ll * n_seqs)));
}

template <typename T, int D>
cudaError_t launch_d(const CacheAttnArgs& a, cudaStream_t stream) {
  switch (row_eights(a.H, a.c.Hkv, a.c.T, a.c.n_seqs)) {
    case 1: return launch_t<T, D, 1>(a, stream);
    case 2: return launch_t<T, D, 2>(a, stream);
    case 3: return launch_t<T, D, 3>(a, stream);
    case 4: return launch_t<T, D, 4>(a, stream);
    default: return launch_cache_tile(a, stream);
  }
}

template <int D, int NT>
size_t workspace_t(int sms) {
  return 2ull * sms * Layout<D, NT>::kPerSm * Layout<D, NT>::kPartial * sizeof(float);
}

template <int D>
size_t workspace_d(int eights, int sms) {
  switch (eights) {
    case 1: return workspace_t<D, 1>(sms);
    case 2: return workspace_t<D, 2>(sms);
    case 3: return workspace_t<D, 3>(sms);
    case 4: return workspace_t<D, 4>(sms);
    default: return cache_tile_workspace(D, sms);
  }
}

}  // namespace

// A workspace for T rows of a batch serves every smaller T: the kernels of fewer rows have more CTAs on a
// multiprocessor, and with D = 64 that of 9 to 16 rows needs more than that of 17 to 24.
size_t cache_attention_workspace(int H, int Hkv, int D, int T, int n_seqs, int sms) {
  const int eights = row_eights(H, Hkv, T, n_seqs);
  size_t most = eights == 0 ? cache_tile_workspace(D, sms) : 0;
  for (int e = 1; e <= (eights == 0 ? 4 : eights); ++e) {
    most = std::max(most, D == 64 ? workspace_d<64>(e, sms) : workspace_d<128>(e, sms));
  }
  return most;
}

cudaError_t launch_cache_attention(const CacheAttnArgs& a, cudaStream_t stream) {
  if (a.dtype == FA_DTYPE_F16) {
    return a.D == 64 ? launch_d<__half, 64>(a, stream) : launch_d<__half, 128>(a, stream);
  }
  return a.D == 64 ? launch_d<__nv_bfloat16, 64>(a, stream)
                   : launch_d<__nv_bfloat16, 128>(a, stream);
}

}  // namespace fa_sm100
