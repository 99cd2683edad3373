// Attention of the newest tokens of every sequence over a paged cache.
//
// Every key and value in reach is read once and meets the few rows (tokens x query heads of its kv head) of one sequence: the kernels are bound
// by memory.  What they have to do is to keep enough loads in flight, and to give every SM the same share of bytes whatever the
// lengths are, which only the device knows.  Measured, 64 sequences of up to 8192 tokens, 8 kv heads of 128, 4 query heads to each: bfloat16 222 - 225 us, 95 %
// of the copy rate; 4 bits 114 us, where the chain of a tile counts (50 %; a warp waits for its own instruction before, with three to a scheduler); float32, 8 sequences, 16 heads of 64, window of 2048, 27.2 us (57 %).
//
// Work.  The walk over the keys of one (sequence, tile of rows, group of kv heads) is an item.  The four warps of a CTA have a kv head each, so that they
// read neighbouring bytes of the same tokens at about the same time (of a 4-bit cache, whose powers of two for 8 heads are one 32-byte sector, 1.8 times the
// bytes came from memory when a CTA had one head), and no results to put together; with two or one head to a CTA, where their number allows no more or items
// are few, two or four warps share one.  An item is cut into units, a tile of keys for every warp.  All units of all items lie on one line, each item's with
// room before them for what it takes to begin and finish an item: 1.5 units with eight rows to a tile, 3 with sixteen, 2 in FMA arithmetic.  (Without it a
// sequence of one token, 8 items to finish, kept its CTA for 9 us after the others.  With 0.5 units in place of these: 128 sequences of up to 256 tokens 27
// us and 23, 32 of up to 8192 with 28 rows 240 and 227, of 4 bits 204 and 182.  With 3 units for eight rows, too,
// 256 sequences of up to 512 take 68 in place of 70, one of 1500 12.3 in place of 11.)  The line is cut into as many even runs as CTAs fit on the chip; a run ends in the middle of an item as a
// rule.  Each CTA finds its run from the lengths.  An item that lies within one run is finished there; the parts of others go to the workspace, at most two
// from a CTA, and paged_join_kernel puts them together in the order of the keys.
//
// Each warp has its own ring of stages in shared memory that it fills by cp.async: no warp waits for another before the end of an item (nor there, with a
// head of its own), and the ring runs on into the next item.  Pages are looked up for every key (any page
// size), a tile ahead of the copy.
//
// Keys outside [lo, hi), which no row of the tile sees, are not read: zeros stand there.  Where the rows of a tile see different keys of a tile of
// keys (several new tokens), each token's rows are multiplied by values that are zero where the token does not see them, so that an infinity or
// a NaN reaches only the rows that see it.
#include <type_traits>

#include "paged.cuh"

namespace bma {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr float kLn2 = 0.6931471805599453f;

struct PagedParams {
  bma_paged_cache c;
  bma_paged_attn_args a;
  int G, rows, row_tiles, entries;     // query heads to a kv head, rows to a kv head, tiles of them, (sequence, tile) pairs
  int heads, heads_log2, splits;       // kv heads to a CTA (1, 2, 4), warps to a head
  int positions;                       // what the page table covers
  int page_shift;                      // log2 of the page size, -1 where that is no power of two
  uint32_t page_units, slot_units, head_units;      // strides of the cache, in 16 bytes
  int scale_words;                     // 4 bits: a head's four powers of two can be read at once, at these strides in words
  uint32_t scale_page, scale_slot, scale_head;
  float scale_log2;
  int* status;
  float* part_o;                       // [2 * CTAs][heads][rows of a tile][DP]
  float2* part_ml;                     // [2 * CTAs][heads][rows of a tile]
  int by_item;                         // meta has a place for every item, else for every CTA, whichever are fewer:
  int4* meta;                          // first CTA with a part of an item (-1: there are no parts to join), slot of its part, CTA with the last part, item
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {     // 16 bytes, or zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_committed() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_awaited() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void matrices(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void matrices_turned(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {      // nothing to add to
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Where a CTA puts the parts of its warps together, in the stages that they have just read: eight rows of a warp at a time, lines of DP + 8 floats; the last
// 8 floats of a line keep the lines in different banks; they hold maximum and sum of rows r and r + 8.
template <int DP>
struct Buffer {
  static constexpr int kLine = DP + 8, kBytes = 8 * kLine * 4;
  uint8_t* at;          // of warp 0
  int stride;           // bytes to the next warp's
  __device__ __forceinline__ float* line(int warp, int r) const { return reinterpret_cast<float*>(at + warp * stride) + r * kLine; }
  __device__ __forceinline__ float2& stat(int warp, int row) const { return *reinterpret_cast<float2*>(line(warp, row & 7) + DP + (row >> 3) * 2); }
};
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// The keys that a tile of rows sees, and who its rows are.
struct Entry {
  int b, row0;             // sequence, first row
  int first, count;        // position of the first new token, number of real ones
  int lo, hi, base;        // keys [lo, hi); the walk starts at `base`
  int units;               // at least 1: an item without keys is written, too
  int t0, t1;              // tokens of the rows, real ones
  int all_from, all_to;    // every row sees keys [all_from, all_to]
  bool one;                // the rows are of one token
  __device__ __forceinline__ bool cut(int k0, int n) const { return k0 < all_from || k0 + n - 1 > all_to; }
};
template <int ROWS, int TILE>
__device__ __forceinline__ Entry entry_of(const PagedParams& p, int e) {
  Entry x;
  x.b = e / p.row_tiles;
  x.row0 = (e - x.b * p.row_tiles) * ROWS;
  const NewTokens n = new_tokens(p.a.lengths, p.a.new_lengths, x.b, p.a.T);
  x.count = n.count;
  x.first = (int)max(n.first, (int64_t)-(1 << 30));
  x.t0 = x.row0 / p.G;
  const int last = (min(x.row0 + ROWS, p.rows) - 1) / p.G;
  x.one = x.t0 == last;
  x.t1 = min(last, x.count - 1);
  x.lo = x.hi = 0;
  if (x.t0 <= x.t1) {
    const int64_t end = n.first + x.t1 + 1;
    x.hi = (int)min(max(end, (int64_t)0), (int64_t)p.positions);
    if (end > p.positions) report_device_error(p.status, kStatusPaged);
    x.lo = p.a.window < 0 ? 0 : (int)min(max(n.first + x.t0 - p.a.window, (int64_t)0), (int64_t)x.hi);
  }
  x.all_to = x.first + x.t0;
  x.all_from = p.a.window < 0 ? x.lo : max(x.lo, (int)max((int64_t)x.first + x.t1 - p.a.window, (int64_t)0));
  x.base = x.lo & ~(TILE - 1);
  x.units = max(1, (x.hi - x.base + p.splits * TILE - 1) / TILE >> (2 - p.heads_log2));      // (of splits * TILE keys)
  return x;
}

// A unit, and its place on the line.
constexpr int kUnit = 2;          // places of a unit
template <int ROWS, int TILE, int ITEM>      // ITEM: places before the units of an item
struct Cursor {
  Entry x;
  int e, h, unit;               // h: this warp's kv head
  int64_t at;
  __device__ __forceinline__ void next(const PagedParams& p) {
    at += kUnit;
    if (++unit < x.units) return;
    at += ITEM;
    unit = 0;
    h += p.heads;
    if (h < p.c.Hkv) return;
    h &= p.heads - 1;
    if (++e < p.entries) x = entry_of<ROWS, TILE>(p, e);
  }
  __device__ __forceinline__ int tile(const PagedParams& p, int warp) const { return x.base + (unit * p.splits + (warp >> p.heads_log2)) * TILE; }
};

// [begin, end) of CTA `cta`'s run
__device__ __forceinline__ int64_t run_begin(int64_t total, int cta, int ctas) { return total * cta / ctas; }

// Where in the cache a key's heads lie, in units of 16 bytes (the host has checked that this fits); none: kNowhere.
constexpr uint32_t kNowhere = 0xffffffffu;
struct Place {
  int page, slot;
  __device__ __forceinline__ void look_up(const PagedParams& p, const Entry& x, int key) {
    page = -1;
    slot = 0;
    if (key >= x.lo && key < x.hi) {
      const int i = p.page_shift < 0 ? key / p.c.page_size : key >> p.page_shift;
      slot = key - i * p.c.page_size;
      page = __ldg(p.c.page_table + (int64_t)x.b * p.c.table_stride + i);
      if (page < 0) page = -2;       // (told from a key that is not looked up)
    }
  }
  __device__ __forceinline__ bool there(const PagedParams& p) const {
    if (page >= 0 && page < p.c.pages) return true;
    if (page != -1) report_device_error(p.status, kStatusPaged);
    return false;
  }
  __device__ __forceinline__ uint32_t at(const PagedParams& p, int h) const {
    return there(p) ? page * p.page_units + slot * p.slot_units + h * p.head_units : kNowhere;
  }
};

__device__ __forceinline__ const __nv_bfloat16* query_row(const PagedParams& p, const Entry& x, int h, int row) {
  return static_cast<const __nv_bfloat16*>(p.a.q.ptr) + x.b * p.a.q.stride_b + (row / p.G) * p.a.q.stride_l + (h * p.G + row % p.G) * p.a.q.stride_h;
}

// Statistics and masks of a warp's rows: scores lie in the accumulators as [keys, rows], and this lane's rows are 2t and 2t + 1 of each of NT tiles of 8.
template <int NT>
struct Rows {
  float m[NT][2], l[NT][2];    // maximum so far (log2 units), this lane's share of the sum
  int at[NT][2];               // position of the row's token; below every key where it is not real
  __device__ __forceinline__ void start(const PagedParams& p, const Entry& x, int lane) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int row = x.row0 + i * 8 + (lane & 3) * 2 + s, t = row / p.G;
        at[i][s] = row < p.rows && t < x.count ? x.first + t : -1;
        m[i][s] = -INFINITY;
        l[i][s] = 0.f;
      }
  }
  __device__ __forceinline__ bool sees(const PagedParams& p, int i, int s, int key) const {
    return key <= at[i][s] && (p.a.window < 0 || key >= at[i][s] - p.a.window);
  }
  // Takes this lane's maxima to those of the rows, and what has been added up (o, a column for each row) to the new ones; `top` becomes what exponents
  // are taken against, 2^up below the maximum.
  template <int N>
  __device__ __forceinline__ void rescale(int i, float (&top)[2], float (&o)[N][4], float up = 0.f) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int b = 4; b < 32; b <<= 1) top[s] = fmaxf(top[s], __shfl_xor_sync(0xffffffffu, top[s], b));
    if (__any_sync(0xffffffffu, top[0] != m[i][0] || top[1] != m[i][1])) {
      float f[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        f[s] = top[s] == -INFINITY ? 1.f : exp2_approx(m[i][s] - top[s]);
        l[i][s] *= f[s];
        m[i][s] = top[s];
      }
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] *= f[e & 1];
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) top[s] = top[s] == -INFINITY ? 0.f : top[s] - up;
  }
  template <int DP>
  __device__ __forceinline__ void stats(const Buffer<DP>& buffer, int warp, int lane, float up = 0.f) const {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float x = l[i][s];
#pragma unroll
        for (int b = 4; b < 32; b <<= 1) x += __shfl_xor_sync(0xffffffffu, x, b);
        if (lane < 4) buffer.stat(warp, i * 8 + lane * 2 + s) = make_float2(m[i][s] - up, x);
      }
  }
};
// Halves of a pair of keys that the token at `at` sees, as a mask of 16-bit values
__device__ __forceinline__ uint32_t seen_pair(const PagedParams& p, int at, int key) {
  uint32_t m = 0;
  if (key <= at && (p.a.window < 0 || key >= at - p.a.window)) m |= 0xffffu;
  if (key + 1 <= at && (p.a.window < 0 || key + 1 >= at - p.a.window)) m |= 0xffff0000u;
  return m;
}
// At the beginning of a branch that is rarely taken: without it the compiler runs both ways and selects, for every tile.
__device__ __forceinline__ void rarely() { asm volatile("" ::: "memory"); }
// An 8 x 8 matrix of 16-bit values, [keys, rows], turned
__device__ __forceinline__ uint32_t turned(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Copies of a tile's rows of BYTES bytes (16 * CHUNKS), keys to `to`, values SIDE further on; `mine` is the place of this lane's key (lane % TILE), SLOT(r, chunk) where
// chunk `chunk` of row r goes.
template <int TILE, int CHUNKS, int SIDE, typename F>
__device__ __forceinline__ void copy_rows(const PagedParams& p, uint32_t mine, int chunks, uint32_t to, int lane, F slot) {
  constexpr int kAtOnce = 32 / CHUNKS;       // rows copied by one instruction
  const int chunk = lane % CHUNKS;
  const char* k = static_cast<const char*>(p.c.k) + chunk * 16;
  const char* v = static_cast<const char*>(p.c.v) + chunk * 16;
  if (__all_sync(0xffffffffu, mine != kNowhere) && chunks == CHUNKS) {
#pragma unroll
    for (int i = 0; i < TILE / kAtOnce; ++i) {
      const int r = i * kAtOnce + lane / CHUNKS;
      const int64_t from = (int64_t)__shfl_sync(0xffffffffu, mine, r) * 16;
      const uint32_t dst = to + slot(r, chunk);
      copy16(dst, k + from, true);
      copy16(dst + SIDE, v + from, true);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < TILE / kAtOnce; ++i) {
    const int r = i * kAtOnce + lane / CHUNKS;
    const uint32_t at = __shfl_sync(0xffffffffu, mine, r);
    const bool there = at != kNowhere && chunk < chunks;
    const int64_t from = there ? (int64_t)at * 16 : -(int64_t)chunk * 16;
    const uint32_t dst = to + slot(r, chunk);
    copy16(dst, k + from, there);
    copy16(dst + SIDE, v + from, there);
  }
}

// ---- bfloat16: matrix instructions fed by ldmatrix ------------------------------------------------------------------
// Keys are the M of mma.m16n8k16 and rows (tokens x heads) its N for the scores; components are the M and rows the N for the sums: 8 rows are a
// tile, where rows as M would make 16 of one.  The weights go from the accumulators of the one to the operand of the other by movmatrix, as two bfloat16 numbers each,
// the first cut off and the second what is left, with 2^-20 of the weight added: both are above zero for weights down to 2^-106, so that an infinite value stays one.  Together they are good
// to 2^-15: rounded to one, they were the largest error of a call (2^-8; bfloat16 results were 14 - 34 % further off
// than their own rounding makes them).  That costs 0.4 % for the serving batch, whose time is the memory's, 3 % with 16 rows to a kv head, 5 % with 28.
template <int DP, int NT>
struct CoreBf16 {
  static constexpr int kDP = DP, kRows = NT * 8, kTile = 16, kItem = NT == 1 ? 3 : 6, kStages = DP == 128 ? (NT == 1 ? 2 : 3) : 4, kMinCtas = NT == 1 ? 3 : 2;      // (two stages and three CTAs 220 us, three and two 238: 64 sequences of up to 8192)
  static constexpr int kRowBytes = DP * 2, kSide = kTile * kRowBytes, kStageBytes = 2 * kSide, kExtra = 0;
  using Cur = Cursor<kRows, kTile, kItem>;

  uint32_t q[NT][DP / 16][2];
  float o[NT][DP / 16][4];
  Rows<NT> rows;
  Place place;

  __device__ __forceinline__ void prepare(uint8_t*) {}
  __device__ __forceinline__ void look_up(const PagedParams& p, const Cur& c, int warp, int lane) { place.look_up(p, c.x, c.tile(p, warp) + (lane & 15)); }
  __device__ __forceinline__ void settle(uint8_t*) {}
  __device__ __forceinline__ void issue(const PagedParams& p, const Cur& c, uint8_t* smem, int stage, int lane) {
    copy_rows<kTile, DP / 8, kSide>(p, place.at(p, c.h), p.c.d / 8, smem_at(smem) + stage, lane, [](int r, int chunk) { return r * kRowBytes + ((chunk ^ (r & 7)) << 4); });
  }
  __device__ __forceinline__ void begin(const PagedParams& p, const Cur& c, int lane) {
    const int g = lane >> 2, t = lane & 3;
    rows.start(p, c.x, lane);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int row = c.x.row0 + i * 8 + g;
      const __nv_bfloat16* from = query_row(p, c.x, c.h, min(row, p.rows - 1));
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int d = k * 16 + u * 8 + 2 * t;
          q[i][k][u] = row < p.rows && d < p.c.d ? __ldg(reinterpret_cast<const uint32_t*>(from + d)) : 0u;
        }
#pragma unroll
      for (int j = 0; j < DP / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][j][e] = 0.f;
    }
  }
  __device__ __forceinline__ void take(const PagedParams& p, const Cur& c, const uint8_t* stage, int k0, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const uint32_t ks = smem_at(stage), vs = ks + kSide;
    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
    {
      const int r = lane & 15, half = lane >> 4;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        uint32_t a[4];
        matrices(a, ks + r * kRowBytes + (((2 * k + half) ^ (r & 7)) << 4));
#pragma unroll
        for (int i = 0; i < NT; ++i) mma_bf16(s[i], a, q[i][k][0], q[i][k][1]);
      }
    }
    const bool cut = c.x.cut(k0, kTile);
    constexpr float kUp = 1.f + 1.f / (1 << 20);
    uint32_t w[NT][2], rest[NT][2];      // weights, and what is left of them
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float top[2] = {rows.m[i][0], rows.m[i][1]};
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] *= p.scale_log2;
      if (cut) {
        rarely();
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!rows.sees(p, i, e & 1, k0 + (e >> 1) * 8 + g)) s[i][e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) top[e & 1] = fmaxf(top[e & 1], s[i][e]);
      rows.rescale(i, top, o[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = exp2_approx(s[i][e] - top[e & 1]);
        rows.l[i][e & 1] += s[i][e];
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t x = __float_as_uint(s[i][2 * u]), y = __float_as_uint(s[i][2 * u + 1]);
        const __nv_bfloat162 low = __floats2bfloat162_rn(fmaf(s[i][2 * u], kUp, -__uint_as_float(x & 0xffff0000u)), fmaf(s[i][2 * u + 1], kUp, -__uint_as_float(y & 0xffff0000u)));
        w[i][u] = turned(__byte_perm(x, y, 0x7632));
        rest[i][u] = turned(*reinterpret_cast<const uint32_t*>(&low));
      }
    }
    const int r = ((lane >> 4) << 3) + (lane & 7), second = (lane >> 3) & 1;
    if (!cut || c.x.one) {
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) {
        uint32_t a[4];
        matrices_turned(a, vs + r * kRowBytes + (((2 * j + second) ^ (r & 7)) << 4));
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          mma_bf16(o[i][j], a, w[i][0], w[i][1]);
          mma_bf16(o[i][j], a, rest[i][0], rest[i][1]);
        }
      }
      return;
    }
    for (int tok = c.x.t0; tok <= c.x.t1; ++tok) {
      const int at = c.x.first + tok;
      const uint32_t seen[2] = {seen_pair(p, at, k0 + 2 * t), seen_pair(p, at, k0 + 8 + 2 * t)};
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) {
        uint32_t a[4];
        matrices_turned(a, vs + r * kRowBytes + (((2 * j + second) ^ (r & 7)) << 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] &= seen[e >> 1];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float x[4] = {0.f, 0.f, 0.f, 0.f};
          mma_bf16(x, a, w[i][0], w[i][1]);
          mma_bf16(x, a, rest[i][0], rest[i][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (rows.at[i][e & 1] == at) o[i][j][e] += x[e];
        }
      }
    }
  }
  __device__ __forceinline__ void stats(const Buffer<DP>& buffer, int warp, int lane) const { rows.stats(buffer, warp, lane); }
  // Rows [8 pass, 8 pass + 8) times factor(row) into lines
  template <typename F>
  __device__ __forceinline__ void put(int pass, F factor, float* out, int lane) const {
    const int g = lane >> 2, t = lane & 3;
    const float f[2] = {factor(pass * 8 + 2 * t), factor(pass * 8 + 2 * t + 1)};
#pragma unroll
    for (int i = 0; i < NT; ++i)
      if (pass == i) {
#pragma unroll
        for (int j = 0; j < DP / 16; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) out[(2 * t + (e & 1)) * Buffer<DP>::kLine + j * 16 + (e >> 1) * 8 + g] = o[i][j][e] * f[e & 1];
      }
  }
};

// ---- 4 bits: the same products in float16 -----------------------------------------------------------------------------
// Codes become float16 as they are, and products of codes are exact; the powers of two join elsewhere.  Keys: a k-step of the instruction lies within 32
// components, whose sum is multiplied by their power in float32.  Values: of a head's powers the largest, 2^E, is taken out and joins the exponent of the weight;
// what remains, 2^(e - E) from 2^-14 to 1, multiplies the weights of each 32 components.  The running maximum is over score + E, so that the weights that go through
// float16 are at most 1, and the sum of weights takes 2^-E back out.  Rows of Q are brought to at most 2^15 by a power of two (what float16 holds: their components
// count to 2^-40 of the row's largest).  Weights are held times 2^15, too: they are good to 2^-11 of themselves
// down to 2^-29 of the row's largest, and to 2^-40 of that below, where their products with 2^(e - E) are rounded once more.
//
// That holds as long as E is between -40 and 40 (with one maximum for both, a weight 2^-126 below it is lost to the sum of weights, whose key may be the only one
// of ordinary values) and no power of a head lies 2^14 below its largest.  Powers of 2^-103 and less count as zeros: they are what heads of zeros have.  From a tile of keys on
// that breaks this (`far`), a warp takes its item as take_wide does: maximum and sum of weights as without powers, the products of every 32
// components with maxima of their own.  There a component is as good as if its group of 32 stood alone, for any powers.  (All tiles taken so: 64 sequences of up to 8192 tokens,
// 8 kv heads of 128, 187 us in place of 114, one of 131072, four tokens, 138 in place of 78.)
//
// Where components lie among those of a k-step, or of a tile of the sums, is free as long as both operands agree: ldmatrix hands each lane four codes of 32 components
// (turned: of two keys), and they are taken in the order in which they come.
template <int DP, int NT>
struct Core4bit {
  static constexpr int kDP = DP, kRows = NT * 8, kTile = 32, kItem = NT == 1 ? 3 : 6, kStages = 2, kMinCtas = NT > 1 ? 2 : DP == 64 ? 4 : 3;
  static constexpr int kRowBytes = DP / 2, kSide = kTile * kRowBytes, kGroups = DP / 32;
  // after keys and values: powers of keys [32][4] (float32), of values [4][32] (float16, by key_of's rows), E and 2^-E of values [32][2], bytes of their powers [32] (take_wide's)
  static constexpr int kKeyPowers = 2 * kSide, kValuePowers = kKeyPowers + 512, kTops = kValuePowers + 256, kBytes = kTops + 256, kStageBytes = kBytes + 128, kExtra = 0;
  static_assert(kStages == 2, "`far` is that of the tile taken next");
  static constexpr float kWeightUp = 15.f;
  static constexpr float kWideUp = -24.f;      // take_wide: sums of weights times values of 2^127 overflow from 2^24 keys on
  static constexpr int kLeastTop = 127 - 40, kMostTop = 127 + 40, kSpread = 14, kZero = 127 - 103, kMostKey = 127 + 100;
  using Cur = Cursor<kRows, kTile, kItem>;

  uint32_t q[NT][DP / 16][2];
  float o[NT][DP / 16][4];
  float scale[NT][2];
  Rows<NT> rows;
  Place place;
  uint32_t k_bytes, v_bytes;    // the powers of two of this lane's key of the last tile issued
  int pending;                  // and where its stage lies, negative where there is none
  bool far, wide;               // the last tile settled, and this item from some tile on, are take_wide's

  __device__ __forceinline__ void prepare(uint8_t*) { pending = -1; wide = false; }
  __device__ __forceinline__ void look_up(const PagedParams& p, const Cur& c, int warp, int lane) { place.look_up(p, c.x, c.tile(p, warp) + lane); }
  // 16-byte chunks of a row are permuted so that 8 rows of a chunk lie in different banks
  static __device__ __forceinline__ int chunk_at(int r, int chunk) { return r * kRowBytes + ((DP == 128 ? chunk ^ (r >> 1 & 3) : chunk ^ (r >> 2 & 1)) << 4); }

  __device__ __forceinline__ void issue(const PagedParams& p, const Cur& c, uint8_t* smem, int stage, int lane) {
    settle(smem);
    const uint32_t mine = place.at(p, c.h);
    k_bytes = v_bytes = 0;       // (of a key that is not read: zeros)
    if (mine != kNowhere) {
      if (p.scale_words) {
        const uint32_t word = place.page * p.scale_page + place.slot * p.scale_slot + c.h * p.scale_head;
        k_bytes = __ldg(reinterpret_cast<const uint32_t*>(p.c.k_scale) + word);
        v_bytes = __ldg(reinterpret_cast<const uint32_t*>(p.c.v_scale) + word);
      } else {
        rarely();
        const int64_t at = (int64_t)place.page * p.c.scale_stride_page + (int64_t)place.slot * p.c.scale_stride_slot + (int64_t)c.h * p.c.scale_stride_head;
        const int n = p.c.d / 32;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < kGroups && i < n) {
            k_bytes |= (uint32_t)__ldg(p.c.k_scale + at + i) << (8 * i);
            v_bytes |= (uint32_t)__ldg(p.c.v_scale + at + i) << (8 * i);
          } else {                                           // (no components there)
            k_bytes |= (k_bytes & 255) << (8 * i);
            v_bytes |= (v_bytes & 255) << (8 * i);
          }
      }
    }
    pending = stage;
    copy_rows<kTile, DP / 32, kSide>(p, mine, p.c.d / 32, smem_at(smem) + stage, lane, [](int r, int chunk) { return chunk_at(r, chunk); });
  }
  // The powers of two that were asked for with the last tile, into its stage.
  __device__ __forceinline__ void settle(uint8_t* smem) {
    if (pending < 0) return;
    uint8_t* to = smem + pending;
    const int lane = threadIdx.x & 31;
    const int b[4] = {(int)(v_bytes & 255), (int)(v_bytes >> 8 & 255), (int)(v_bytes >> 16 & 255), (int)(v_bytes >> 24)};
    int top = max(max(b[0], b[1]), max(b[2], b[3]));
    const int least = min(min(b[0], b[1]), min(b[2], b[3]));
    // a byte of a key that is 0 or above kMostKey (top bits: it borrows, or it carries)
    const uint32_t odd_key = (((k_bytes - 0x01010101u) & ~k_bytes) | (((k_bytes & 0x7f7f7f7fu) + (255 - kMostKey) * 0x01010101u) & k_bytes)) & 0x80808080u;
    const bool rare = top > kMostTop || least < max(top, kLeastTop) - kSpread || odd_key;
    top = max(top, kLeastTop);
    uint32_t f[4];      // 2^(e - E) as float16
    float kp[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = b[i] * 1024 + (15 - top) * 1024;
      kp[i] = __uint_as_float((i == 0 ? k_bytes << 23 : i == 1 ? k_bytes << 15 : i == 2 ? k_bytes << 7 : k_bytes >> 1) & 0x7f800000u);
    }
    far = false;
    if (__any_sync(0xffffffffu, rare)) {
      rarely();
      top = kLeastTop;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = b[i] == 255 ? top : max(top, b[i]);
      bool mine = top > kMostTop;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int x = b[i] - top + 15;
        mine |= b[i] > kZero && x < 15 - kSpread;
        f[i] = b[i] == 255 ? 0x7fff : x >= 15 - kSpread ? x << 10 : 0;
        const int key = k_bytes >> (8 * i) & 255;
        mine |= key > kMostKey && key != 255;
        kp[i] = e8m0_value(key);
      }
      far = __any_sync(0xffffffffu, mine);
    }
    if (far || wide) *reinterpret_cast<uint32_t*>(to + kBytes + lane * 4) = v_bytes;
    uint16_t* vp = reinterpret_cast<uint16_t*>(to + kValuePowers) + (lane & 16) + (lane & 6) + (lane >> 3 & 1) + (lane & 1) * 8;      // the row m of the key
#pragma unroll
    for (int i = 0; i < kGroups; ++i) vp[i * 32] = (uint16_t)f[i];
    *reinterpret_cast<float4*>(to + kKeyPowers + lane * 16) = make_float4(kp[0], kp[1], kp[2], kp[3]);
    *reinterpret_cast<float2*>(to + kTops + lane * 8) = make_float2((float)(top - 127), __uint_as_float((uint32_t)(254 - top) << 23));
    pending = -1;
  }
  __device__ __forceinline__ void begin(const PagedParams& p, const Cur& c, int lane) {
    const int g = lane >> 2, t = lane & 3;
    wide = false;
    rows.start(p, c.x, lane);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int row = c.x.row0 + i * 8 + g;
      const __nv_bfloat16* from = query_row(p, c.x, c.h, min(row, p.rows - 1));
      float x[kGroups][8];       // components 8t and up of each 32
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        const int d = k * 32 + t * 8;
        const uint4 v = row < p.rows && d < p.c.d ? __ldg(reinterpret_cast<const uint4*>(from + d)) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int z = 0; z < 8; ++z) {
          x[k][z] = __uint_as_float(z & 1 ? w[z / 2] & 0xffff0000u : w[z / 2] << 16);
          top = fmaxf(top, fabsf(x[k][z]));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(max((int)(__float_as_uint(top) >> 23), 15), 254);      // top < 2^(e - 126)
      const float down = __uint_as_float((uint32_t)(268 - e) << 23), up = p.scale_log2 * __uint_as_float((uint32_t)(e - 14) << 23);
      scale[i][0] = __shfl_sync(0xffffffffu, up, t * 8);                      // (row 2t is that of lanes 8t to 8t + 3)
      scale[i][1] = __shfl_sync(0xffffffffu, up, t * 8 + 4);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int z = (k & 1) * 4 + u * 2;
          const __half2 h = __floats2half2_rn(x[k / 2][z] * down, x[k / 2][z + 1] * down);
          q[i][k][u] = *reinterpret_cast<const uint32_t*>(&h);
        }
#pragma unroll
      for (int j = 0; j < DP / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][j][e] = 0.f;
    }
  }
  static __device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  // The key of row m of a tile of 16: so that the values' codes of keys m = 2t and 2t + 8, which the sums want in one register, lie in neighbouring keys.
  static __device__ __forceinline__ int key_of(int m) { return (m & 1) * 8 + (m & 6) + (m >> 3); }
  // Scores of keys 16 h and up: s[i][e] for key key_of((e >> 1) * 8 + g), row 2t + (e & 1).  SCALED: with the row's scale (which comes first there: powers of keys may
  // be as large as a float32 is)
  template <bool SCALED>
  __device__ __forceinline__ void scores(const uint8_t* stage, int h, int lane, float (&s)[NT][4]) const {
    const int g = lane >> 2;
    uint32_t w[2][kGroups];      // codes of keys g and g + 8
    if constexpr (DP == 128) {
#pragma unroll
      for (int u = 0; u < 2; ++u) matrices(w[u], smem_at(stage) + chunk_at(h * 16 + key_of(u * 8 + (lane & 7)), lane >> 3));
    } else {
      uint32_t x[4];
      matrices(x, smem_at(stage) + chunk_at(h * 16 + key_of((lane >> 4) * 8 + (lane & 7)), lane >> 3 & 1));
      w[0][0] = x[0]; w[0][1] = x[1]; w[1][0] = x[2]; w[1][1] = x[3];
    }
    float f[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float4 x = *reinterpret_cast<const float4*>(stage + kKeyPowers + (h * 16 + key_of(u * 8 + g)) * 16);
      f[u][0] = x.x; f[u][1] = x.y; f[u][2] = x.z; f[u][3] = x.w;
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      uint32_t x[4], y[4];
      from_e2m1x8(w[0][k], x);
      from_e2m1x8(w[1][k], y);
      const uint32_t a[2][4] = {{x[0], y[0], x[1], y[1]}, {x[2], y[2], x[3], y[3]}};
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        float z[4];
        mma_f16_first(z, a[0], q[i][2 * k][0], q[i][2 * k][1]);
        mma_f16(z, a[1], q[i][2 * k + 1][0], q[i][2 * k + 1][1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (SCALED) z[e] *= scale[i][e & 1];
          s[i][e] = k ? fmaf(z[e], f[e >> 1][k], s[i][e]) : z[e] * f[e >> 1][k];
        }
      }
    }
  }
  __device__ __forceinline__ void take(const PagedParams& p, const Cur& c, const uint8_t* stage, int k0, int lane) {
    if (far || wide) {
      rarely();
      take_wide(p, c, stage, k0, lane);
      return;
    }
    const int g = lane >> 2;
    const bool cut = c.x.cut(k0, kTile);
    float s[2][NT][4];
    scores<false>(stage, 0, lane, s[0]);
    scores<false>(stage, 1, lane, s[1]);
    float2 tops[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int u = 0; u < 2; ++u) tops[h][u] = *reinterpret_cast<const float2*>(stage + kTops + (h * 16 + key_of(u * 8 + g)) * 8);
    uint32_t w[2][NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float top[2] = {rows.m[i][0], rows.m[i][1]};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[h][i][e] = fmaf(s[h][i][e], scale[i][e & 1], tops[h][e >> 1].x);
      if (cut) {
        rarely();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!rows.sees(p, i, e & 1, k0 + h * 16 + key_of((e >> 1) * 8 + g))) s[h][i][e] = -INFINITY;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) top[e & 1] = fmaxf(top[e & 1], s[h][i][e]);
      rows.rescale(i, top, o[i], kWeightUp);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[h][i][e] = exp2_approx(s[h][i][e] - top[e & 1]);
          rows.l[i][e & 1] = fmaf(s[h][i][e], tops[h][e >> 1].y, rows.l[i][e & 1]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const __half2 x = __floats2half2_rn(s[h][i][2 * u], s[h][i][2 * u + 1]);
          w[h][i][u] = turned(*reinterpret_cast<const uint32_t*>(&x));
        }
      }
    }
    if (!cut || c.x.one) {
      values<false>(p, stage, k0, 0, lane, w[0], 0);
      values<false>(p, stage, k0, 1, lane, w[1], 0);
    } else
      for (int tok = c.x.t0; tok <= c.x.t1; ++tok) {
        values<true>(p, stage, k0, 0, lane, w[0], c.x.first + tok);
        values<true>(p, stage, k0, 1, lane, w[1], c.x.first + tok);
      }
  }
  // The codes of keys 16 h and up, of components 32 k to 32 k + 63: four of keys 2t and 2t + 1 (rows m = 2t and 2t + 8 of the tile), and of keys 8 further on (m = 2t + 1 and 2t + 9)
  static __device__ __forceinline__ void codes(const uint8_t* stage, int h, int k, int lane, uint32_t (&x)[2][2]) {
    uint32_t y[4];
    matrices_turned(y, smem_at(stage) + kSide + chunk_at(h * 16 + (lane >> 3 & 1) * 8 + (lane & 7), k + (lane >> 4)));
    x[0][0] = y[0]; x[0][1] = y[1]; x[1][0] = y[2]; x[1][1] = y[3];
  }
  // and as operands: a byte for each pair of keys and component
  static __device__ __forceinline__ void operands(const uint32_t (&x)[2], uint32_t (&a)[2][4]) {
    uint32_t even[4], odd[4];
    from_e2m1x8((x[0] & 0x0f0f0f0fu) | ((x[1] * 16u) & 0xf0f0f0f0u), even);                      // components 0 and 2 of four, of rows m = 2t; of 2t + 8
    from_e2m1x8((__umulhi(x[0], 1u << 28) & 0x0f0f0f0fu) | (x[1] & 0xf0f0f0f0u), odd);           // (a shift by the multiplier, which has time)
#pragma unroll
    for (int j = 0; j < 2; ++j) { a[j][0] = even[j]; a[j][1] = odd[j]; a[j][2] = even[j + 2]; a[j][3] = odd[j + 2]; }
  }
  // The same tile whatever its powers: o += V^T (weight times power), for every 32 components against the tile's own maximum of that.  From here on o and l are in
  // units of 2^(m - kWideUp), m the maximum of the scores.
  __device__ __forceinline__ void take_wide(const PagedParams& p, const Cur& c, const uint8_t* stage, int k0, int lane) {
    const int g = lane >> 2;
    if (!wide) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int z = 0; z < 2; ++z) rows.m[i][z] += kWideUp - kWeightUp;      // (the same units: m need not be the maximum, only near it)
      wide = true;
    }
    float s[2][NT][4];
    scores<true>(stage, 0, lane, s[0]);
    scores<true>(stage, 1, lane, s[1]);
    uint32_t bytes[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int u = 0; u < 2; ++u) bytes[h][u] = *reinterpret_cast<const uint32_t*>(stage + kBytes + (h * 16 + key_of(u * 8 + g)) * 4);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float top[2] = {rows.m[i][0], rows.m[i][1]};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!rows.sees(p, i, e & 1, k0 + h * 16 + key_of((e >> 1) * 8 + g))) s[h][i][e] = -INFINITY;
          top[e & 1] = fmaxf(top[e & 1], s[h][i][e]);
        }
      rows.rescale(i, top, o[i], kWideUp);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) rows.l[i][e & 1] += exp2_approx(s[h][i][e] - top[e & 1]);
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        float x[2][4], most[2] = {-INFINITY, -INFINITY}, f[2], acc[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int b = bytes[h][e >> 1] >> (8 * k) & 255;
            x[h][e] = s[h][i][e] == -INFINITY ? -INFINITY : s[h][i][e] + (b == 255 ? __uint_as_float(0x7fffffffu) : (float)(b - 127));
            most[e & 1] = fmaxf(most[e & 1], x[h][e]);
          }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
#pragma unroll
          for (int lanes = 4; lanes < 32; lanes <<= 1) most[z] = fmaxf(most[z], __shfl_xor_sync(0xffffffffu, most[z], lanes));
          const bool none = most[z] == -INFINITY;                 // (there `top` says nothing of what the factor may be)
          most[z] = none ? 0.f : most[z] - kWeightUp;
          f[z] = none ? 0.f : exp2_approx(0.5f * (most[z] - top[z]));          // (twice: the product may be below 2^-126)
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t b[2], y[2][2], a[2][4];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const __half2 w = __floats2half2_rn(exp2_approx(x[h][2 * u] - most[0]), exp2_approx(x[h][2 * u + 1] - most[1]));
            b[u] = turned(*reinterpret_cast<const uint32_t*>(&w));
          }
          codes(stage, h, k & ~1, lane, y);
          operands(y[k & 1], a);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (h == 0) mma_f16_first(acc[j], a[j], b[0], b[1]);
            else mma_f16(acc[j], a[j], b[0], b[1]);
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][2 * k + j][e] = fmaf(acc[j][e] * f[e & 1], f[e & 1], o[i][2 * k + j][e]);
      }
    }
  }
  // o += V^T w over keys 16 h and up.  ONE: only the rows of the token at `at`, of the keys that it sees.
  template <bool ONE>
  __device__ __forceinline__ void values(const PagedParams& p, const uint8_t* stage, int k0, int h, int lane, const uint32_t (&w)[NT][2], int at) {
    const int t = lane & 3;
    uint32_t x[kGroups / 2][2][2];
#pragma unroll
    for (int k = 0; k < kGroups; k += 2) codes(stage, h, k, lane, x[k / 2]);
    uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
    if (ONE) {
      const uint32_t a = seen_pair(p, at, k0 + h * 16 + 2 * t), b = seen_pair(p, at, k0 + h * 16 + 8 + 2 * t);
      seen[0] = __byte_perm(a, b, 0x5410);
      seen[1] = __byte_perm(a, b, 0x7632);
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const uint32_t f0 = *reinterpret_cast<const uint32_t*>(stage + kValuePowers + (k * 32 + h * 16 + 2 * t) * 2);
      const uint32_t f1 = *reinterpret_cast<const uint32_t*>(stage + kValuePowers + (k * 32 + h * 16 + 8 + 2 * t) * 2);
      uint32_t a[2][4];
      operands(x[k / 2][k & 1], a);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        uint32_t b0 = times(w[i][0], f0), b1 = times(w[i][1], f1);
        if (ONE) { b0 &= seen[0]; b1 &= seen[1]; }          // (weight and power: a value that is not seen may be NaN by its power alone)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (!ONE) mma_f16(o[i][2 * k + j], a[j], b0, b1);
          else {
            float z[4];
            mma_f16_first(z, a[j], b0, b1);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (rows.at[i][e & 1] == at) o[i][2 * k + j][e] += z[e];
          }
        }
      }
    }
  }
  __device__ __forceinline__ void stats(const Buffer<DP>& buffer, int warp, int lane) const { rows.stats(buffer, warp, lane, wide ? kWideUp : kWeightUp); }
  template <typename F>
  __device__ __forceinline__ void put(int pass, F factor, float* out, int lane) const {
    const int g = lane >> 2, t = lane & 3;
    const float f[2] = {factor(pass * 8 + 2 * t), factor(pass * 8 + 2 * t + 1)};
#pragma unroll
    for (int i = 0; i < NT; ++i)
      if (pass == i) {
#pragma unroll
        for (int k = 0; k < kGroups; ++k)
#pragma unroll
          for (int s = 0; s < 2; ++s)
            *reinterpret_cast<float4*>(out + (2 * t + s) * Buffer<DP>::kLine + k * 32 + g * 4) =
                make_float4(o[i][2 * k][s] * f[s], o[i][2 * k][2 + s] * f[s], o[i][2 * k + 1][s] * f[s], o[i][2 * k + 1][2 + s] * f[s]);
      }
  }
};

// ---- float32: FMA arithmetic ----------------------------------------------------------------------------------------------
// For the scores two or four lanes share a key, for the sums a lane has DP / 32 columns; the rows of Q are read from shared memory, by all lanes at once.
template <int DP, int ROWS>
struct CoreF32 {
  static constexpr int kDP = DP, kRows = ROWS, kTile = DP == 128 ? 8 : 16, kItem = 4, kStages = 2, kMinCtas = ROWS <= 4 ? 3 : 2;
  static constexpr int kRowBytes = DP * 4, kSide = kTile * kRowBytes, kStageBytes = 2 * kSide;
  static constexpr int kParts = 32 / kTile, kChunks = DP / 4 / kParts;      // lanes to a key, 16-byte chunks to each of them
  static constexpr int kQRow = DP + 4 * kParts;      // floats: each part of a row lies 4 further on than the one before would have it, in other banks
  static constexpr int kExtra = kWarps * (ROWS * kQRow + kTile * ROWS) * 4;
  static constexpr int kCols = DP / 32;
  using Cur = Cursor<kRows, kTile, kItem>;

  static constexpr int kOwn = ROWS >= kParts ? ROWS / kParts : ROWS;      // rows whose softmax a lane takes: a key's lanes share them out, where there are enough

  float o[ROWS][kCols];
  float m[kOwn], l[kOwn];      // of the lane's rows; l: its key's share
  int own;                     // the first of them
  Place place;
  float *qs, *ps;

  __device__ __forceinline__ void prepare(uint8_t* extra) {
    qs = reinterpret_cast<float*>(extra) + (threadIdx.x >> 5) * (ROWS * kQRow + kTile * ROWS);
    ps = qs + ROWS * kQRow;
  }
  __device__ __forceinline__ void look_up(const PagedParams& p, const Cur& c, int warp, int lane) { place.look_up(p, c.x, c.tile(p, warp) + (lane & (kTile - 1))); }
  __device__ __forceinline__ void settle(uint8_t*) {}
  __device__ __forceinline__ void issue(const PagedParams& p, const Cur& c, uint8_t* smem, int stage, int lane) {
    copy_rows<kTile, DP / 4, kSide>(p, place.at(p, c.h), p.c.d / 4, smem_at(smem) + stage, lane, [](int r, int chunk) { return r * kRowBytes + ((chunk ^ (r & 7)) << 4); });
  }
  __device__ __forceinline__ void begin(const PagedParams& p, const Cur& c, int lane) {
    // All of the rows are asked for before one is put down: CTAs with many short items are the last to end.  (A value at a time, and `finish` with the statistics
    // of a row for every value: 16 sequences of up to 4096 tokens, 4 kv heads of 128, 16 rows to each 231 us, so 73; 8 kv heads, 4 rows 125 and 58.)
    constexpr int kLanes = DP / 4, kAtOnce = 32 / kLanes;       // lanes to a row, rows at a time
    const int n = min(ROWS, p.rows - c.x.row0), d = lane % kLanes * 4;
    float4 x[(ROWS + kAtOnce - 1) / kAtOnce];
#pragma unroll
    for (int r0 = 0; r0 < ROWS; r0 += kAtOnce) {
      const int r = r0 + lane / kLanes, row = c.x.row0 + r, t = row / p.G;
      x[r0 / kAtOnce] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < n && d < p.c.d)
        x[r0 / kAtOnce] = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.a.q.ptr) + c.x.b * p.a.q.stride_b + t * p.a.q.stride_l +
                                                                (c.h * p.G + row - t * p.G) * p.a.q.stride_h + d));
    }
    __syncwarp();                // (the last item's rows have been read)
#pragma unroll
    for (int r0 = 0; r0 < ROWS; r0 += kAtOnce)
      if (r0 + lane / kLanes < ROWS) *reinterpret_cast<float4*>(qs + (r0 + lane / kLanes) * kQRow + d + d / (4 * kChunks) * 4) = x[r0 / kAtOnce];
    __syncwarp();
    own = 0;
    if (ROWS >= kParts) {        // halves of the rows, then quarters: as they are handed out in `take`
      int n = ROWS;
#pragma unroll
      for (int b = 16; b >= kTile; b >>= 1) own += lane & b ? (n >>= 1) : (n >>= 1, 0);
    }
#pragma unroll
    for (int r = 0; r < kOwn; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int j = 0; j < kCols; ++j) o[r][j] = 0.f;
  }
  __device__ __forceinline__ void take(const PagedParams& p, const Cur& c, const uint8_t* stage, int k0, int lane) {
    const int key = lane & (kTile - 1), part = lane / kTile;
    float s[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) s[r] = 0.f;
#pragma unroll 4
    for (int i = 0; i < kChunks; ++i) {
      const int chunk = part * kChunks + i;
      const float4 k = *reinterpret_cast<const float4*>(stage + key * kRowBytes + ((chunk ^ (key & 7)) << 4));
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float4 x = *reinterpret_cast<const float4*>(qs + r * kQRow + chunk * 4 + part * 4);
        s[r] = fmaf(x.x, k.x, fmaf(x.y, k.y, fmaf(x.z, k.z, fmaf(x.w, k.w, s[r]))));
      }
    }
    // The lanes of a key add up their parts of its products; each ends with its own rows.
    if constexpr (ROWS >= kParts) {
      int n = ROWS;
#pragma unroll
      for (int b = 16; b >= kTile; b >>= 1) {
        n >>= 1;
        const bool upper = lane & b;
#pragma unroll
        for (int r = 0; r < ROWS / 2; ++r)
          if (r < n) {
            const float give = upper ? s[r] : s[r + n], keep = upper ? s[r + n] : s[r];
            s[r] = keep + __shfl_xor_sync(0xffffffffu, give, b);
          }
      }
    } else {
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int b = kTile; b < 32; b <<= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], b);
    }
    const bool cut = c.x.cut(k0, kTile), strict = cut && p.a.T > 1;      // strict: some row sees what another does not
    float f[kOwn];
    bool moved = false;
#pragma unroll
    for (int r = 0; r < kOwn; ++r) {
      float x = s[r] * p.scale_log2;
      bool seen = true;
      if (cut) {
        rarely();
        const int row = c.x.row0 + own + r, t = row / p.G, at = row < p.rows && t < c.x.count ? c.x.first + t : -1, k = k0 + key;
        seen = k <= at && (p.a.window < 0 || k >= at - p.a.window);
        if (!seen) x = -INFINITY;
      }
      float top = fmaxf(m[r], x);
#pragma unroll
      for (int b = 1; b < kTile; b <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
      const float base = top == -INFINITY ? 0.f : top;
      f[r] = top == m[r] ? 1.f : exp2_approx(m[r] - base);
      moved |= top != m[r];
      m[r] = top;
      x = exp2_approx(x - base);
      l[r] = fmaf(l[r], f[r], x);
      if (ROWS >= kParts || part == 0) ps[key * ROWS + own + r] = seen ? x : strict ? -1.f : 0.f;
    }
    if (__any_sync(0xffffffffu, moved)) {
      // what has been added up, to the new maxima; row r is that of the lanes of key 0 that own it
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        float g = f[r % kOwn];
        if (ROWS >= kParts) {
          int from = 0, n = ROWS, q = r;
#pragma unroll
          for (int b = 16; b >= kTile; b >>= 1) {
            n >>= 1;
            if (q >= n) { from |= b; q -= n; }
          }
          g = __shfl_sync(0xffffffffu, f[q], from);
        }
#pragma unroll
        for (int j = 0; j < kCols; ++j) o[r][j] *= g;
      }
    }
    __syncwarp();
#pragma unroll 4
    for (int k = 0; k < kTile; ++k) {
      float v[kCols];
      const uint8_t* row = stage + kSide + k * kRowBytes;
      if constexpr (kCols == 4) {
        const float4 x = *reinterpret_cast<const float4*>(row + ((lane ^ (k & 7)) << 4));
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(row + (((lane >> 1) ^ (k & 7)) << 4) + (lane & 1) * 8);
        v[0] = x.x; v[1] = x.y;
      }
      constexpr int kAtOnce = ROWS < 4 ? ROWS : 4;
#pragma unroll
      for (int r4 = 0; r4 < ROWS; r4 += kAtOnce) {
        float w[4];
        if constexpr (ROWS == 1) w[0] = ps[k];
        else {
          const float4 w4 = *reinterpret_cast<const float4*>(ps + k * ROWS + r4);
          w[0] = w4.x; w[1] = w4.y; w[2] = w4.z; w[3] = w4.w;
        }
#pragma unroll
        for (int r = 0; r < kAtOnce; ++r)
#pragma unroll
          for (int j = 0; j < kCols; ++j) {
            if (strict && w[r] == -1.f) continue;
            o[r4 + r][j] = fmaf(w[r], v[j], o[r4 + r][j]);
          }
      }
    }
    __syncwarp();
  }
  __device__ __forceinline__ void stats(const Buffer<DP>& buffer, int warp, int lane) const {
#pragma unroll
    for (int r = 0; r < kOwn; ++r) {
      float x = l[r];
#pragma unroll
      for (int b = 1; b < kTile; b <<= 1) x += __shfl_xor_sync(0xffffffffu, x, b);
      if (ROWS >= kParts ? (lane & (kTile - 1)) == 0 : lane == 0) buffer.stat(warp, own + r) = make_float2(m[r], x);
    }
  }
  template <typename F>
  __device__ __forceinline__ void put(int pass, F factor, float* out, int lane) const {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r >> 3 == pass) {
        const float f = factor(r);
#pragma unroll
        for (int j = 0; j < kCols; ++j) out[(r & 7) * Buffer<DP>::kLine + lane * kCols + j] = o[r][j] * f;
      }
  }
};

// ---- the walk ---------------------------------------------------------------------------------------------------------------
template <class Core>
constexpr int paged_smem() {
  static_assert(Core::kStageBytes >= Buffer<Core::kDP>::kBytes && Core::kStageBytes % 16 == 0, "a warp's rows fit into a stage");
  constexpr int bytes = kWarps * Core::kStages * Core::kStageBytes + Core::kExtra;
  static_assert(Core::kMinCtas * (bytes + 1024) <= 228 * 1024, "the CTAs that plan_paged counts on fit an SM's shared memory");
  return bytes;
}

// A finished row's value: four components and (at the first) the log-sum-exp; zeros for a token that is not real.
__device__ __forceinline__ void write_result(const PagedParams& p, int b, int h, int row, bool real, int col, float4 x, float top, float sum) {
  const bool any = real && (sum > 0.f || sum != sum);
  const float f = any ? 1.f / sum : 0.f;
  x = any ? make_float4(x.x * f, x.y * f, x.z * f, x.w * f) : make_float4(0.f, 0.f, 0.f, 0.f);
  const int t = row / p.G, head = h * p.G + row % p.G;
  const int64_t at = b * p.a.o.stride_b + t * p.a.o.stride_l + head * p.a.o.stride_h + col;
  if (col < p.c.d) {
    if (p.a.o.dtype == BMA_DTYPE_F32) *reinterpret_cast<float4*>(static_cast<float*>(p.a.o.ptr) + at) = x;
    else {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x, x.y), hi = __floats2bfloat162_rn(x.z, x.w);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.a.o.ptr) + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
  if (col == 0 && p.a.lse) p.a.lse[((int64_t)b * p.a.Hq + head) * p.a.T + t] = any ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
}

// A head's item, of one warp or put together from those that share the head: written as the result where the CTA has all of it, else as a part.
template <class Core>
__device__ __forceinline__ void finish(const PagedParams& p, Core& core, const typename Core::Cur& c, bool whole, int slot, const Buffer<Core::kDP>& buffer, int warp, int lane) {
  constexpr int DP = Core::kDP;
  const auto meet = [&] {
    if (p.splits == 1) __syncwarp();
    else __syncthreads();
  };
  const int mine = warp & (p.heads - 1), of_head = (warp >> p.heads_log2) * 32 + lane;      // this warp's head of the CTA's; the thread among those of the head
  core.stats(buffer, warp, lane);
  meet();
  const int n = min(Core::kRows, p.rows - c.x.row0);
  for (int pass = 0; pass * 8 < n; ++pass) {
    // statistics of the warps that share the head, a row to a lane (and again in every 8 lanes)
    const int of_lane = pass * 8 + (lane & 7);
    float top = -INFINITY, sum = 0.f;
    for (int w = mine; w < kWarps; w += p.heads) top = fmaxf(top, buffer.stat(w, of_lane).x);
    const float base = top == -INFINITY ? 0.f : top, factor = exp2_approx(buffer.stat(warp, of_lane).x - base);
    for (int w = mine; w < kWarps; w += p.heads) {
      const float2 x = buffer.stat(w, of_lane);
      sum = fmaf(x.y, exp2_approx(x.x - base), sum);
    }
    core.put(pass, [&](int row) { return __shfl_sync(0xffffffffu, factor, row & 7); }, buffer.line(warp, 0), lane);
    meet();
    for (int i = of_head; i < 8 * (DP / 4); i += p.splits * 32) {
      const int r = i / (DP / 4), col = i % (DP / 4) * 4, row = pass * 8 + r;
      const float row_top = __shfl_sync(0xffffffffu, top, r), row_sum = __shfl_sync(0xffffffffu, sum, r);
      if (row >= n) continue;
      float4 x = *reinterpret_cast<const float4*>(buffer.line(mine, r) + col);
      for (int w = mine + p.heads; w < kWarps; w += p.heads) {
        const float4 y = *reinterpret_cast<const float4*>(buffer.line(w, r) + col);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      }
      if (!whole) {
        const int64_t at = ((int64_t)slot * p.heads + mine) * Core::kRows + row;
        *reinterpret_cast<float4*>(p.part_o + at * DP + col) = x;
        if (col == 0) p.part_ml[at] = make_float2(row_top, row_sum);
      } else write_result(p, c.x.b, c.h, c.x.row0 + row, (c.x.row0 + row) / p.G < c.x.count, col, x, row_top, row_sum);
    }
    meet();
  }
}

template <class Core>
__global__ void __launch_bounds__(kThreads, Core::kMinCtas) paged_kernel(const __grid_constant__ PagedParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  using Cur = typename Core::Cur;
  constexpr int NS = Core::kStages;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;");

  // The run of this CTA: prefix sums of the entries' units, kThreads at a time.
  int64_t* scan = reinterpret_cast<int64_t*>(smem);      // sums of the warps, then the entry that the run begins in, and where
  auto block_scan = [&](int x, int64_t& before, int64_t& all) {
    int64_t y = x;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    if (lane == 31) scan[warp] = y;
    __syncthreads();
    before = y - x;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      all += scan[w];
    }
    __syncthreads();
  };
  auto places_of = [&](int e) { return e < p.entries ? Core::kItem + kUnit * entry_of<Core::kRows, Core::kTile>(p, e).units : 0; };
  int64_t total = 0, before = 0, all = 0;
  int own = 0;
  for (int e0 = 0; e0 < p.entries; e0 += kThreads) {
    own = places_of(e0 + threadIdx.x);
    block_scan(own, before, all);
    total += all;
  }
  const int groups = p.c.Hkv >> p.heads_log2;
  total *= groups;
  if (threadIdx.x == 0 && !p.by_item) p.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
  const int ctas = (int)min((int64_t)gridDim.x, max(total / kUnit, (int64_t)1));       // (within an item every run has a unit's beginning)
  if (blockIdx.x >= ctas) return;
  const int64_t begin = run_begin(total, blockIdx.x, ctas), end = run_begin(total, blockIdx.x + 1, ctas);
  int64_t gone = 0;
  for (int e0 = 0; e0 < p.entries; e0 += kThreads) {
    if (p.entries > kThreads) {
      own = places_of(e0 + threadIdx.x);
      block_scan(own, before, all);
    }
    const int64_t from = (gone + before) * groups;
    if (begin >= from && begin < from + (int64_t)own * groups) {
      scan[kWarps + 1] = e0 + threadIdx.x;
      scan[kWarps + 2] = begin - from;
    }
    gone += all;
  }
  __syncthreads();
  Cur next;
  next.e = (int)scan[kWarps + 1];
  const int64_t within = scan[kWarps + 2];
  next.x = entry_of<Core::kRows, Core::kTile>(p, next.e);
  const int places = Core::kItem + kUnit * next.x.units;
  const int group = (int)(within / places);
  const int inside = (int)(within - (int64_t)group * places);                       // of the item
  next.h = group * p.heads + (warp & (p.heads - 1));
  next.unit = max(inside - Core::kItem + kUnit - 1, 0) / kUnit;                           // the first unit that begins in the run
  next.at = begin - inside + Core::kItem + kUnit * next.unit;
  if (next.unit >= next.x.units) {                                                  // (that is the next item's)
    --next.unit;
    next.at -= kUnit;
    next.next(p);
  }
  __syncthreads();              // (copies go there next)

  Core core;
  core.prepare(smem + kWarps * NS * Core::kStageBytes);
  Cur here = next;
  if (here.at >= end) return;  // (a place before an item's units is all there is)
  core.look_up(p, next, warp, lane);
  int to = 0, from = 0;        // stages to fill and to read next
  auto issue = [&] {
    if (next.at < end) {
      core.issue(p, next, smem, (warp * NS + to) * Core::kStageBytes, lane);
      to = to == NS - 1 ? 0 : to + 1;
      next.next(p);
      if (next.at < end) core.look_up(p, next, warp, lane);
    }
    copies_committed();
  };
  for (int i = 0; i < NS - 1; ++i) issue();
  bool fresh = true;           // the first unit of an item in this run
  int first_unit = here.unit;
  bool first_item = true;
  while (here.at < end) {
    core.settle(smem);
    issue();
    if (fresh) {                 // (its queries come while the keys do)
      core.begin(p, here, lane);
      first_unit = here.unit;
      fresh = false;
    }
    copies_awaited<NS - 1>();
    __syncwarp();
    const int k0 = here.tile(p, warp);
    if (k0 < here.x.hi) core.take(p, here, smem + (warp * NS + from) * Core::kStageBytes, k0, lane);
    __syncwarp();
    const bool last = here.unit + 1 == here.x.units;
    if (last || here.at + kUnit >= end) {
      const bool whole = last && first_unit == 0;
      const int slot = 2 * blockIdx.x + (first_item ? 0 : 1);
      if (first_unit == 0 && threadIdx.x == 0) {        // the first part of an item, or all of it
        const int item = here.e * groups + (here.h >> p.heads_log2);
        if (!whole) {
          const int64_t item_end = here.at + kUnit * (here.x.units - 1 - here.unit) + 1;   // one past where its last unit begins
          int cta = (int)((item_end - 1) * ctas / total);             // the CTA whose run holds that
          while (run_begin(total, cta + 1, ctas) < item_end) ++cta;
          while (run_begin(total, cta, ctas) >= item_end) --cta;
          p.meta[p.by_item ? item : blockIdx.x] = make_int4(blockIdx.x, slot, cta, item);
        } else if (p.by_item) p.meta[item] = make_int4(-1, 0, 0, 0);
      }
      const Buffer<Core::kDP> buffer{smem + from * Core::kStageBytes, NS * Core::kStageBytes};
      finish<Core>(p, core, here, whole, slot, buffer, warp, lane);
      fresh = true;
      first_item = false;
    }
    here.next(p);
    from = from == NS - 1 ? 0 : from + 1;
  }
  copies_awaited<0>();
}

// A row of a head of an item that several CTAs had parts of.
template <int ROWS>
struct Joined {
  int4 m;                        // (of PagedParams::meta)
  int b, head, mine, row, of_sequence, parts, heads;
  bool real;
  // Row and head `of_item` of the item of this CTA; false: there are no parts, or no such row.
  __device__ __forceinline__ bool open(const PagedParams& p, int of_item) {
    m = p.meta[blockIdx.x];
    if (m.x < 0) return false;
    heads = p.heads;
    mine = of_item & (p.heads - 1);
    row = of_item >> p.heads_log2;
    const int groups = p.c.Hkv >> p.heads_log2, e = m.w / groups;
    head = (m.w - e * groups) * p.heads + mine;
    b = e / p.row_tiles;
    const int row0 = (e - b * p.row_tiles) * ROWS;
    of_sequence = row0 + row;
    if (row >= min(ROWS, p.rows - row0)) return false;
    real = of_sequence / p.G < new_tokens(p.a.lengths, p.a.new_lengths, b, p.a.T).count;
    parts = m.z - m.x + 1;
    return true;
  }
  __device__ __forceinline__ int64_t slot(int i) const { return ((int64_t)(i == 0 ? m.y : 2 * (m.x + i)) * heads + mine) * ROWS + row; }      // of part i
};

// One CTA: a row, its warps taking parts in turn.
template <int DP, int ROWS>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(const __grid_constant__ PagedParams p) {
  __shared__ float4 sums[kWarps][DP / 4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Joined<ROWS> of;
  if (!of.open(p, blockIdx.y)) return;
  // Parts 32 at a time, all that is read of them at once: their statistics by every warp, a part to a lane, their sums by the warps in turn.
  float top = -INFINITY, sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < of.parts; i0 += 32) {
    const float2 ml = i0 + lane < of.parts ? p.part_ml[of.slot(i0 + lane)] : make_float2(-INFINITY, 0.f);
    float4 y[32 / kWarps];
#pragma unroll
    for (int k = 0; k < 32 / kWarps; ++k) {
      const int i = i0 + k * kWarps + warp;
      y[k] = i < of.parts && lane * 4 < DP ? *reinterpret_cast<const float4*>(p.part_o + of.slot(i) * DP + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float t = ml.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
    t = fmaxf(t, top);
    const float base = t == -INFINITY ? 0.f : t, f = exp2_approx(ml.x - base), g = top == t ? 1.f : exp2_approx(top - base);
    top = t;
    sum = fmaf(sum, g, ml.y * f);
    x.x *= g; x.y *= g; x.z *= g; x.w *= g;
#pragma unroll
    for (int k = 0; k < 32 / kWarps; ++k) {
      const float fi = __shfl_sync(0xffffffffu, f, k * kWarps + warp);
      x.x = fmaf(y[k].x, fi, x.x); x.y = fmaf(y[k].y, fi, x.y); x.z = fmaf(y[k].z, fi, x.z); x.w = fmaf(y[k].w, fi, x.w);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane * 4 < DP) sums[warp][lane] = x;
  __syncthreads();
  if (warp || lane * 4 >= DP) return;
#pragma unroll
  for (int w = 1; w < kWarps; ++w) {
    const float4 y = sums[w][lane];
    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
  }
  write_result(p, of.b, of.head, of.of_sequence, of.real, lane * 4, x, top, sum);
}

// The same where most items have few parts: a warp to a row.
template <int DP, int ROWS>
__global__ void __launch_bounds__(kThreads) paged_join_few_kernel(const __grid_constant__ PagedParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  Joined<ROWS> of;
  if (!of.open(p, blockIdx.y * kWarps + (threadIdx.x >> 5))) return;
  float top = -INFINITY, sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  auto take = [&](int i0, auto at_once) {       // parts i0 and up, all that is read of them at once
    constexpr int N = decltype(at_once)::value;
    float2 ml[N];
    float4 y[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const bool in = i0 + k < of.parts;
      ml[k] = in ? p.part_ml[of.slot(i0 + k)] : make_float2(-INFINITY, 0.f);
      y[k] = in && lane * 4 < DP ? *reinterpret_cast<const float4*>(p.part_o + of.slot(i0 + k) * DP + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float t = top;
#pragma unroll
    for (int k = 0; k < N; ++k) t = fmaxf(t, ml[k].x);
    const float base = t == -INFINITY ? 0.f : t, g = top == t ? 1.f : exp2_approx(top - base);
    top = t;
    sum *= g;
    x.x *= g; x.y *= g; x.z *= g; x.w *= g;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float f = exp2_approx(ml[k].x - base);
      sum = fmaf(ml[k].y, f, sum);
      x.x = fmaf(y[k].x, f, x.x); x.y = fmaf(y[k].y, f, x.y); x.z = fmaf(y[k].z, f, x.z); x.w = fmaf(y[k].w, f, x.w);
    }
  };
  if (of.parts <= 4) take(0, std::integral_constant<int, 4>());
  else
    for (int i0 = 0; i0 < of.parts; i0 += 16) take(i0, std::integral_constant<int, 16>());      // a long sequence among many short ones
  if (lane * 4 < DP) write_result(p, of.b, of.head, of.of_sequence, of.real, lane * 4, x, top, sum);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
int validate_paged(const bma_paged_cache* c, const bma_paged_attn_args* a) {
  int rc = validate_cache(c);
  if (rc != BMA_OK) return rc;
  BMA_REQUIRE(a && a->T > 0 && a->Hq > 0 && a->lengths, BMA_ERR_ARG);
  BMA_REQUIRE(a->Hq % c->Hkv == 0, BMA_ERR_ARG);
  BMA_REQUIRE(a->Hq <= 65535 && (int64_t)a->T * a->Hq < (1ll << 30), BMA_ERR_LIMIT);
  BMA_REQUIRE(a->q.dtype == (c->dtype == BMA_DTYPE_F32 ? BMA_DTYPE_F32 : BMA_DTYPE_BF16), BMA_ERR_UNSUPPORTED);
  BMA_REQUIRE(a->o.dtype == BMA_DTYPE_F32 || a->o.dtype == BMA_DTYPE_BF16, BMA_ERR_UNSUPPORTED);
  // the kernels count in 16 bytes
  const int64_t bytes = c->dtype == BMA_DTYPE_F32 ? 4 : c->dtype == BMA_DTYPE_BF16 ? 2 : 1;
  const int64_t last = ((int64_t)(c->pages - 1) * c->stride_page + (int64_t)(c->page_size - 1) * c->stride_slot + (int64_t)(c->Hkv - 1) * c->stride_head) * bytes / 16;
  BMA_REQUIRE(last < (int64_t)kNowhere, BMA_ERR_LIMIT);
  return BMA_OK;
}

struct PagedLaunch {
  int rows_of_tile, dp, tile, ctas_per_sm, heads;
  int ctas, entries, row_tiles, groups;
  int metas() const { return (int)std::min<int64_t>(ctas, (int64_t)entries * groups); }
  size_t bytes() const { return (size_t)ctas * 2 * heads * rows_of_tile * (dp * 4 + 8) + (size_t)metas() * 16; }
};

// The instance for a call: heads of up to 64 or 128 components; tiles of as many rows as the call has, up to 16: more do not leave room for the sums in
// registers (32 sequences of up to 8192 tokens with 28 rows to a kv head of 128, bfloat16, 353 us in one tile of 32, 257 in two of 16, the second of which finds
// the keys in the L2).
// As many CTAs as run at once, or as there can be units.
bool plan_paged(const bma_paged_cache& c, const bma_paged_attn_args& a, PagedLaunch& l) {
  const int rows = a.T * (a.Hq / c.Hkv);
  l.dp = c.d <= 64 ? 64 : 128;
  l.tile = c.dtype == BMA_DTYPE_MXFP4 ? 32 : c.dtype == BMA_DTYPE_F32 && l.dp == 128 ? 8 : 16;
  l.rows_of_tile = c.dtype == BMA_DTYPE_F32 && rows <= 4 ? (rows == 1 ? 1 : 4) : rows <= 8 ? 8 : 16;
  // (what registers and shared memory allow; the kMinCtas of the instances)
  l.ctas_per_sm = c.dtype == BMA_DTYPE_F32 ? (l.rows_of_tile <= 4 ? 3 : 2) : l.rows_of_tile > 8 ? 2 : c.dtype == BMA_DTYPE_MXFP4 && l.dp == 64 ? 4 : 3;
  l.row_tiles = ceil_div(rows, l.rows_of_tile);
  const int64_t entries = (int64_t)c.B * l.row_tiles;
  if (entries >= (1 << 30)) return false;
  l.entries = (int)entries;
  // Heads to a CTA: as many as there are warps, as long as the CTAs do not get more than 8 parts of an item.  (64 sequences of up to 8192 tokens, 8 kv heads of 128, 128
  // items for 444 CTAs: 4 bits 119 us with four heads, 140 with one, bfloat16 225 and 224; one sequence of 131072, four tokens, 2 or 8 items for 296 CTAs: 92 and 81,
  // for four times the parts.)
  const int64_t at_once = (int64_t)device_sms(current_device()) * l.ctas_per_sm;
  l.heads = c.Hkv % 4 == 0 ? 4 : c.Hkv % 2 == 0 ? 2 : 1;
  if (entries * (c.Hkv / l.heads) * 8 < at_once) l.heads = 1;
  const int64_t keys = kWarps / l.heads * l.tile;      // of a unit
  l.groups = c.Hkv / l.heads;
  if (entries * l.groups >= (1ll << 31)) return false;
  const int64_t units = entries * l.groups * (((int64_t)c.width * c.page_size + keys - 1) / keys + 1);
  l.ctas = (int)std::min<int64_t>(at_once, units);
  return true;
}

template <class Core>
int launch_paged(const PagedParams& p, const PagedLaunch& l, cudaStream_t st) {
  constexpr int smem = paged_smem<Core>();
  static std::atomic<bool> allowed[kMaxDevices] = {};        // of this instance, by device
  std::atomic<bool>& set = allowed[current_device()];
  if (!set.load(std::memory_order_relaxed)) {
    BMA_CUDA_TRY(cudaFuncSetAttribute(paged_kernel<Core>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    set.store(true, std::memory_order_relaxed);
  }
  paged_kernel<Core><<<l.ctas, kThreads, smem, st>>>(p);
  BMA_CUDA_TRY(cudaGetLastError());
  // Where the average item has fewer than four parts a row to a warp, else to a CTA.  (8 kv heads of 128, bfloat16: 128 sequences of up to 256 tokens, 256 items for 444
  // CTAs, 6 us less; 256 of up to 512 7 less; 32 of up to 8192 with 28 rows, 128 items for 296 CTAs, 8 less, with 16 rows, 64 items, 3 more.  One long
  // sequence among many short ones has many parts, and pays for that: 32768 tokens among 299 of 100 7 more.)
  const int rows = std::min(Core::kRows, p.rows) * p.heads;
  const bool few = (int64_t)l.entries * l.groups * 3 > l.ctas;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(l.metas(), few ? ceil_div(rows, kWarps) : rows);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;      // (its CTAs come up while the last parts are written)
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (few) BMA_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_join_few_kernel<Core::kDP, Core::kRows>, p));
  else BMA_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_join_kernel<Core::kDP, Core::kRows>, p));
  count_launches(2);
  return BMA_OK;
}

template <int DP>
int dispatch_paged(const PagedParams& p, const PagedLaunch& l, cudaStream_t st) {
  switch (p.c.dtype) {
    case BMA_DTYPE_F32:
      if (l.rows_of_tile == 1) return launch_paged<CoreF32<DP, 1>>(p, l, st);
      if (l.rows_of_tile == 4) return launch_paged<CoreF32<DP, 4>>(p, l, st);
      if (l.rows_of_tile == 8) return launch_paged<CoreF32<DP, 8>>(p, l, st);
      return launch_paged<CoreF32<DP, 16>>(p, l, st);
    case BMA_DTYPE_BF16:
      if (l.rows_of_tile == 8) return launch_paged<CoreBf16<DP, 1>>(p, l, st);
      return launch_paged<CoreBf16<DP, 2>>(p, l, st);
    default:
      if (l.rows_of_tile == 8) return launch_paged<Core4bit<DP, 1>>(p, l, st);
      return launch_paged<Core4bit<DP, 2>>(p, l, st);
  }
}

}  // namespace
}  // namespace bma

using namespace bma;

extern "C" {

size_t bma_paged_attn_workspace_bytes(const bma_paged_cache* cache, const bma_paged_attn_args* args) {
  PagedLaunch l;
  return validate_paged(cache, args) == BMA_OK && plan_paged(*cache, *args, l) ? l.bytes() : 0;
}

int bma_paged_attn(const bma_paged_cache* cache, const bma_paged_attn_args* args, void* workspace, size_t workspace_bytes, bma_stream_t stream) {
  int rc = validate_paged(cache, args);
  if (rc != BMA_OK) return rc;
  BMA_REQUIRE(args->q.ptr && args->o.ptr, BMA_ERR_ARG);
  for (const bma_tensor* t : {&args->q, &args->o}) {            // rows start on 16 bytes
    const int vec = t->dtype == BMA_DTYPE_F32 ? 4 : 8;
    BMA_REQUIRE((reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && t->stride_b % vec == 0 && t->stride_l % vec == 0 && t->stride_h % vec == 0, BMA_ERR_UNSUPPORTED);
  }
  PagedLaunch l;
  BMA_REQUIRE(plan_paged(*cache, *args, l), BMA_ERR_LIMIT);
  BMA_REQUIRE(workspace && workspace_bytes >= l.bytes() && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, BMA_ERR_WORKSPACE);
  PagedParams p{};
  p.c = *cache;
  p.a = *args;
  p.G = args->Hq / cache->Hkv;
  p.rows = args->T * p.G;
  p.row_tiles = l.row_tiles;
  p.entries = l.entries;
  p.by_item = (int64_t)l.entries * l.groups <= l.ctas;
  p.heads = l.heads;
  p.heads_log2 = l.heads / 2;
  p.splits = kWarps / l.heads;
  p.positions = cache->width * cache->page_size;
  const int64_t bytes = cache->dtype == BMA_DTYPE_F32 ? 4 : cache->dtype == BMA_DTYPE_BF16 ? 2 : 1;      // (their products fit 32 bits: validate_paged)
  p.page_units = (uint32_t)(cache->stride_page * bytes / 16);
  p.slot_units = (uint32_t)(cache->stride_slot * bytes / 16);
  p.head_units = (uint32_t)(cache->stride_head * bytes / 16);
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (cache->page_size == 1 << i) p.page_shift = i;
  const int64_t last_scale = (int64_t)(cache->pages - 1) * cache->scale_stride_page + (int64_t)(cache->page_size - 1) * cache->scale_stride_slot +
                             (int64_t)(cache->Hkv - 1) * cache->scale_stride_head;
  p.scale_words = cache->dtype == BMA_DTYPE_MXFP4 && cache->d == 128 && last_scale / 4 < (int64_t)kNowhere &&
                  ((reinterpret_cast<uintptr_t>(cache->k_scale) | reinterpret_cast<uintptr_t>(cache->v_scale) | (uintptr_t)cache->scale_stride_page |
                    (uintptr_t)cache->scale_stride_slot | (uintptr_t)cache->scale_stride_head) & 3) == 0;
  p.scale_page = (uint32_t)(cache->scale_stride_page / 4);
  p.scale_slot = (uint32_t)(cache->scale_stride_slot / 4);
  p.scale_head = (uint32_t)(cache->scale_stride_head / 4);
  p.scale_log2 = args->scale * kLog2e;
  BMA_REQUIRE((p.status = device_status_ptr()) != nullptr, BMA_ERR_CUDA);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)2 * l.ctas * l.heads * l.rows_of_tile * l.dp);
  p.meta = reinterpret_cast<int4*>(p.part_ml + (size_t)2 * l.ctas * l.heads * l.rows_of_tile);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return l.dp == 64 ? dispatch_paged<64>(p, l, st) : dispatch_paged<128>(p, l, st);
}

}
