// Attention of one new token over its sequence in a paged KV cache and the depth rows of earlier layers.
//
// For a sequence b and KV head h the G query heads see one list of keys: the sequence's rows (through the
// block table), then the depth rows.  With s_j = scale q . k_j:  o = sum_j 2^(s_j log2 e - m) v_j / l, lse = m + log2 l,
// in one pass with the running maximum m and sum l.  A unit of work has up to kQ = 8 of the G queries, and a key row is read once for them:
// 4 D G flops for 4 D bytes.  More queries are further units, which read the rows again (64 sequences of 4096 rows, 8 heads of
// 128: 172 us with G = 8, 333 with 16, 633 with 32).  So the call is bound by memory, and what the kernel is built for is to
// have bytes on the way at all times:
//
//  - The work, 16-key tiles of every (b, h) in one row, is divided evenly between the CTAs (or their warps) by the lengths on
//    the device (nothing is known on the host, and a captured call must follow new lengths).  A CTA walks its
//    range, which may end one unit, hold several and begin another.  A unit that lies in one CTA's range is
//    written at once, the others' parts are joined by a second, dependent launch.  Where the width of the table says that no
//    sequence is long, all is done in one launch: few units go to a cluster of CTAs each, many short ones to single warps.
//  - A warp takes every fourth tile of a unit's part and copies it, asynchronously, into slots of shared memory of its
//    own, kStages - 1 tiles ahead and across the ends of units: warps do not wait for one another.  An instruction copies
//    whole rows (512 bytes in one piece where a page holds its heads one after another).  Measured on 1 GB: 7.0 TB/s, against
//    5.0 where a lane copies the chunks that it will multiply, eight rows and 64 bytes of each an instruction.
//  - The products are m16n8k16 matrix instructions.  At 16 keys a tile and 8 query rows their rate is far from a
//    limit (32 instructions a tile of 8 KB at D = 128), so that tcgen05 tiles of 128 keys, which need barriers, TMEM and
//    16 times the padding, would buy nothing.  The order of the head's elements within a score is free, and is chosen so
//    that a lane's operands are 16-byte chunks of a row: lane (g, t) = (lane / 4, lane % 4) holds elements 32 j + 8 t .. + 7 of
//    key g.  V is read transposed by the matrix loads.
//  - Eight query rows leave the lower half of the 16-row operand free.  It holds what rounding the upper half to 16
//    bits has left over: the rotated query's remainder (the query is turned here, in 32 bits, without rounding), and that of
//    the probabilities.  So neither is rounded to fewer than 16 significant bits, at no cost.  Against a form that holds 24, 0.3 % of bf16
//    results come out one step away; the error against 64 bits is the same to three digits, as it is the result's own rounding (8
//    bits).  A third part would take half as many score products again, and registers that D = 128 does not have.
//  - In fp16 probabilities are held times 2^15: 65536 keys of 2^-26 beside one of 1 are not to vanish below the type's range.
#pragma once
#include "rotary_kernels.cuh"

namespace moda {
namespace paged {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kTile = 16;          // keys of a warp's step
constexpr int kQ = 8;              // query heads of a unit; more are further units
// A team takes a unit: the four warps of a CTA, which divide its tiles; or, where there are many short units (kShort tiles on average),
// each warp by itself, which has nothing to wait for.  1708 units of one tile, D = 128: 37 us by CTAs, 21 by warps.
constexpr int kShort = 12, kWhole = 2 * kShort;
constexpr int kByWarps = -1;
// Tiles that a unit counts for beyond its own, where the work is divided: beginning and ending one takes a CTA about as long.  37
// sequences of up to 1531 rows, 5 heads of 64 (units of 1 to 97 tiles): 23.2 us without, 18.0 with 4, 16.1 with 8, 16.8 with 16.
__host__ __device__ constexpr int unit_cost(int team) { return team == 1 ? 2 : 8; }
// A range is not made shorter: a unit of two tiles a warp.
__host__ __device__ constexpr int least_places(int team) { return 2 * team + unit_cost(team); }

struct DecodeParams {
  View q, o;                       // [B, G, H, D]
  Pages pages;
  View k, v;                       // [B, 1, H, D]: the new tokens' own rows, which this call writes to the cache (pointers nullptr: none)
  View k_copy, v_copy;             // [B, 1, H, D]: those rows as written once more (pointers nullptr: not)
  int copy_all;                    // also of rows that have no place in the cache (0 without the copies)
  View kd, vd;                     // depth rows (b, layer, h); position p of P lies p * depth_sp further
  int64_t kd_sp, vd_sp;
  const int* depth_positions;      // [B]: positions seen, nullptr: all P
  int P, L;
  FastDiv by_L;
  float* lse;                      // [B, G, H]
  rotary::Args rot;                // of the queries and the own keys, at the last position of the sequence
  int B, H, G;
  float scale_log2;
  int cluster;                     // 0: units are divided evenly over all CTAs; C: each unit over the C CTAs of a cluster; kByWarps: whole units to warps
  // scratch where units are divided over all CTAs
  int2* parts;                     // [kWarps][CTA], of a CTA's one team or four: unit that it begins and others go on with, and how many hold a part
                                   // (none: 0; with four teams the numbers are negative, none: -1)
  int rows;                        // min(G, kQ)
  float2* ml;                      // [team][2][rows]: maximum and sum; part 0 goes on from the team before, part 1 begins here
  float* acc;                      // [team][2][rows][D]
};

template <typename T> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// What the exponents of probabilities are lifted by (the maximum m of a part is the true one less this).
template <typename T> struct Lift { static constexpr float value = 0.f; };
template <> struct Lift<__half> { static constexpr float value = 15.f; };
// Two values as 16 bits each, and what that leaves over.  (A turned fp16 query may be larger than fp16: the upper half is its largest value then.)
template <typename T> __device__ __forceinline__ float largest(float a) { return a; }
template <> __device__ __forceinline__ float largest<__half>(float a) { return isinf(a) ? a : fminf(fmaxf(a, -65504.f), 65504.f); }
template <typename T> __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = Pack<T>::pack(largest<T>(a), largest<T>(b));
  const float2 r = Pack<T>::unpack(hi);
  lo = Pack<T>::pack(a - r.x, b - r.y);
}
// A sum over the two halves.  What is left over is 0 or of either sign: against an infinite key or value it says nothing.
__device__ __forceinline__ float both(float hi, float lo) { return fabsf(lo) < INFINITY ? hi + lo : hi; }
// 16 bytes from global memory to shared memory; !valid: zeros, and nothing is read.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool valid) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" :: "r"(to), "l"(from), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 x;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
  return x;
}

// Four 8 x 8 matrices of 16-bit values, transposed: lane l gives the address of row l % 8 of matrix l / 8, and gets of each matrix the
// elements of column l / 4 in rows 2 (l % 4) and the next.
__device__ __forceinline__ void load_transposed(uint32_t (&x)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
}

__device__ __forceinline__ void sts128(uint32_t at, const uint4& x) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}

// A tile in shared memory: 16 rows of K, 16 of V.  Chunk c (16 bytes) of row r is at place c ^ k_swizzle(r) of its row, or c ^ (r & 7):
// the eight lanes that an access takes together then meet all banks, for the copies (chunks of one row) as for the reads
// (K: chunks 4 j + t of two neighbouring rows g; V: one chunk of eight rows).
template <int D> __host__ __device__ constexpr int stage_bytes() { return kTile * D * 2 * 2; }
__host__ __device__ constexpr int k_swizzle(int r) { return ((r & 1) << 2) | ((r >> 1) & 3); }
constexpr int kStages = 3;
// Rows of 64 elements take half the products and half the registers for them, and nearly as many other instructions a tile: three CTAs an
// SM.  213 sequences of up to 986 rows, 10 heads of 64: 82 us with two (and six stages), 73 with three, 123 with four, whose registers spill.
template <int D> __host__ __device__ constexpr int ctas_per_sm() { return D == 128 ? 2 : 3; }
// The copies' slots and the warps' parts of a unit.  With what the kernel declares statically, two CTAs just fit an SM (D = 128).
template <int D> constexpr size_t smem_bytes() { return (size_t)kWarps * kStages * stage_bytes<D>() + (size_t)kWarps * kQ * D * 4; }
// Four elements from 4 chunk on of a row of those parts; the order of a row's chunks spreads the lanes over the banks.
template <int D> __device__ __forceinline__ float4* part_at(float* parts, int warp, int row, int chunk) {
  return reinterpret_cast<float4*>(parts + (warp * kQ + row) * D) + (chunk ^ row);
}

// Rows in the cache, those with the token's own, depth rows; 16-key tiles of the first two, and of all (at least one).  Depth rows begin a tile.
struct Sequence { int held, len, depth, cached_tiles, tiles; };
__device__ __forceinline__ Sequence sequence(const DecodeParams& p, int b, bool report = false) {
  Sequence s;
  const int len = p.pages.seq_lens[b], seen = p.depth_positions != nullptr ? p.depth_positions[b] : p.P, own = p.k.ptr != nullptr;
  if (report && (len < 0 || len > p.pages.room - own || seen < 0 || seen > p.P)) wrong(kBadLength);
  s.held = min(max(len, 0), p.pages.room);
  s.len = s.held + (len >= 0 && len < p.pages.room ? own : 0);
  s.depth = min(max(seen, 0), p.P) * p.L;
  s.cached_tiles = (s.len + kTile - 1) / kTile;                   // all below 2^31, as the tables are wide
  s.tiles = max(s.cached_tiles + (s.depth + kTile - 1) / kTile, 1);
  return s;
}

// A team's walk over its range: (sequence, unit of it, tiles [t0, t1) of the unit).  A unit takes `cost` places before its tiles.  No
// cost: the range is one of whole units, which are counted (none where a cluster has its one unit).
struct Walk {
  int cost;
  int b, unit;                       // unit: head * query blocks + query block
  Sequence s;
  int t0, t1;
  int64_t left;                      // places (units) of the range behind this unit
  __device__ __forceinline__ int places() const { return s.tiles + cost; }
  // The part of the unit from `place` on.  Short units of single warps stay whole, with the team that has their first place.
  __device__ __forceinline__ void enter(int place) {
    if (cost == 0) {
      --left;
      t0 = 0;
      t1 = s.tiles;
      return;
    }
    const int used = (int)min((int64_t)(places() - place), left);
    left -= used;
    t0 = max(place - cost, 0);
    t1 = max(place + used - cost, 0);
    if (cost == unit_cost(1) && s.tiles <= kWhole) {
      t0 = 0;
      t1 = place == 0 ? s.tiles : 0;
    }
  }
  __device__ __forceinline__ bool next(const DecodeParams& p, int units) {
    if (left <= 0) return false;
    if (++unit == units) {
      unit = 0;
      if (++b >= p.B) return false;  // lengths that another stream changes meanwhile give no right result, but nothing is read outside
      s = sequence(p, b, cost == 0);
    }
    enter(0);
    return t1 > 0;                   // a range may end before the unit's first tile
  }
};

// The places of all units in a row, divided between n teams: team i has [begin(i), begin(i + 1)).
struct Range {
  int64_t each;                      // each, and one more for some: the first `over` are spread over the teams
  uint32_t n, over;
  __device__ __forceinline__ int64_t begin(uint32_t i) const { return each * i + over * i / n; }      // over, i <= n: the product fits
};
__device__ __forceinline__ int64_t quotient(int64_t a, uint32_t b) {            // of numbers that nearly always fit 32 bits
  return (a >> 32) == 0 ? (int64_t)((uint32_t)a / b) : a / b;
}
// The team's size and range, and its walk at the begin of it; at: the place of the walk's unit in the row.  False where there is nothing for it.
__device__ __forceinline__ bool locate(const DecodeParams& p, int units, int* s_tiles, int& team, Range& r, Walk& w, int64_t& at) {
  const int tid = threadIdx.x, lane = tid & 31;
  int sum = 0, before = 0;           // tiles (places) of one unit of each sequence: below 2^31
  int64_t begin = 0, last = 0;       // of this team's range; of the CTA's last team's
  bool passed = false, found = false;      // the place has been; there is a unit for the team
  for (int pass = 0; pass < 2; ++pass)      // adds them up; finds the sequence that holds `begin`
    for (int base = 0; base < p.B; base += kThreads) {
      if (pass == 0 || p.B > kThreads) {
        __syncthreads();
        s_tiles[tid] = base + tid < p.B ? sequence(p, base + tid, pass == 0 && blockIdx.x == 0).tiles : 0;
        __syncthreads();
      }
      int4 x = reinterpret_cast<const int4*>(s_tiles)[lane];
      if (pass == 0) {
        sum += __reduce_add_sync(0xffffffffu, x.x + x.y + x.z + x.w);
        if (base + kThreads < p.B) continue;
        team = (int64_t)p.B * units >= 2 * gridDim.x && sum <= (int64_t)kShort * p.B ? 1 : kWarps;
        w.cost = unit_cost(team);
        const int64_t total = ((int64_t)sum + (int64_t)w.cost * p.B) * units;
        const uint32_t teams = gridDim.x * (kWarps / team), least = least_places(team);
        r.n = (uint32_t)min((int64_t)teams, quotient(total + least - 1, least));
        const uint32_t first = blockIdx.x * (kWarps / team), mine = first + (team == 1 ? tid / 32 : 0);
        if (first >= r.n) return false;
        r.each = quotient(total, r.n);
        r.over = (uint32_t)(total - r.each * r.n);
        last = r.begin(min(first + kWarps / team, r.n) - 1);
        begin = r.begin(min(mine, r.n));
        w.left = mine < r.n ? r.begin(mine + 1) - begin : 0;
        continue;
      }
      if (x.x > 0) x.x += w.cost;    // a sequence has a tile at least
      if (x.y > 0) x.y += w.cost;
      if (x.z > 0) x.z += w.cost;
      if (x.w > 0) x.w += w.cost;
      const int mine = x.x + x.y + x.z + x.w;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const uint32_t here = __ballot_sync(0xffffffffu, begin < (int64_t)(before + incl) * units);
      if (here != 0 && !passed) {
        passed = true;
        const int from = __ffs(here) - 1;
        int first = before + incl - mine, k = 0;      // of the lane's four sequences
        if (begin >= (int64_t)(first + x.x) * units) { first += x.x; k = 1;
          if (begin >= (int64_t)(first + x.y) * units) { first += x.y; k = 2;
            if (begin >= (int64_t)(first + x.z) * units) { first += x.z; k = 3; } } }
        first = __shfl_sync(0xffffffffu, first, from);
        w.b = __shfl_sync(0xffffffffu, base + lane * 4 + k, from);
        w.s = sequence(p, w.b);
        const int64_t off = begin - (int64_t)first * units;
        w.unit = min((int)quotient(off, (uint32_t)w.places()), units - 1);
        const int place = (int)(off - (int64_t)w.unit * w.places());
        at = begin - place;
        w.enter(place);
        found = w.t1 > w.t0;
        if (!found) {                // another team's, or nothing but the places before its tiles
          at += w.places();
          found = w.next(p, units);
        }
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      if (last < (int64_t)before * units) return found;      // the same for all warps, which meet above
    }
  return found;
}
// The same where a cluster of C CTAs has a unit: an even share of its tiles (none for some where there are few).
__device__ __forceinline__ void locate_cluster(const DecodeParams& p, int units, Walk& w) {
  const int id = blockIdx.x / p.cluster, rank = blockIdx.x - id * p.cluster;
  w.b = id / units;
  w.unit = id - w.b * units;
  w.s = sequence(p, w.b, w.unit == 0 && rank == 0 && threadIdx.x == 0);
  w.t0 = (int)((uint32_t)w.s.tiles * rank / p.cluster);           // tiles below 2^27, rank below 16
  w.t1 = (int)((uint32_t)w.s.tiles * (rank + 1) / p.cluster);
  w.left = 0;
  w.cost = 0;
}

// Whole units to warps: an even share of them, no unit being long.  False where there is none for this warp.
__device__ __forceinline__ bool locate_units(const DecodeParams& p, int units, Walk& w) {
  const uint32_t n = gridDim.x * kWarps, i = blockIdx.x * kWarps + threadIdx.x / 32;
  const uint64_t all = (uint64_t)p.B * units;                     // below 2^31, n below 2^16
  const uint32_t begin = (uint32_t)(all * i / n), end = (uint32_t)(all * (i + 1) / n);
  if (begin == end) return false;
  w.b = begin / units;
  w.unit = begin - w.b * units;
  w.s = sequence(p, w.b, w.unit == 0);
  w.cost = 0;
  w.left = end - begin;
  w.enter(0);
  return true;
}

// The new token's own row, row n of a tile that has been copied as it was given: turned there, and written to its place in the cache (page, and slot
// in it) and to the copies.  cs: cosines and sines of its position, which is the queries'.  page < 0: it has no place, and is not seen either: its value
// must not meet the products, where an infinite one would count times 0.
template <typename T, int D>
__device__ __forceinline__ void own_row(const DecodeParams& p, const Walk& w, int h, int page, bool write, uint32_t tile, int n, const float2* cs) {
  constexpr int C = D / 16;
  const int lane = threadIdx.x & 31, c = lane % C;
  if (lane < 2 * C) {
    const bool of_v = lane >= C;
    int c0, c1;
    const bool turns = rotary::item_chunks(p.rot, c, c0, c1) && p.rot.inv_freq != nullptr && !of_v;
    const uint32_t row = tile + (of_v ? kTile + n : n) * D * 2, swizzle = of_v ? n & 7 : k_swizzle(n);
    uint4 x = lds128(row + ((c0 ^ swizzle) << 4)), y = lds128(row + ((c1 ^ swizzle) << 4));
    if (turns) {
      float2 mine[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[i] = cs[8 * c + i];
      rotary::turn<T>(x, y, mine, p.rot.interleaved != 0);
      sts128(row + ((c0 ^ swizzle) << 4), x);
      sts128(row + ((c1 ^ swizzle) << 4), y);
    }
    if (page < 0) {
      sts128(row + ((c0 ^ swizzle) << 4), make_uint4(0, 0, 0, 0));
      sts128(row + ((c1 ^ swizzle) << 4), make_uint4(0, 0, 0, 0));
    }
    if (write && (page >= 0 || p.copy_all != 0)) {
      const int slot = w.s.held - (int)p.pages.by_page.div((uint32_t)w.s.held) * p.pages.page_size;
      const View &to = of_v ? p.pages.v : p.pages.k, &copy = of_v ? p.v_copy : p.k_copy;
      if (page >= 0) {
        *rotary::chunk_at(to, to.off(page, slot, h), c0) = x;
        *rotary::chunk_at(to, to.off(page, slot, h), c1) = y;
      }
      if (copy.ptr != nullptr) {
        *rotary::chunk_at(copy, copy.off(w.b, 0, h), c0) = x;
        *rotary::chunk_at(copy, copy.off(w.b, 0, h), c1) = y;
      }
    }
  }
  __syncwarp();
}

// The own row of a sequence that has no room for it (or whose length is wrong), which is in no tile: into the copies alone.  By one thread; rare.
template <typename T, int D>
__device__ __noinline__ void copy_own_row(const DecodeParams& p, int b, int h, int position) {
#pragma unroll 1
  for (int i = 0; i < 2 * (D / 16); ++i) {
    const bool of_v = i >= D / 16;
    int c0, c1;
    const bool turns = rotary::item_chunks(p.rot, i % (D / 16), c0, c1) && p.rot.inv_freq != nullptr && !of_v;
    const View &from = of_v ? p.v : p.k, &to = of_v ? p.v_copy : p.k_copy;
    uint4 x = *rotary::chunk_at(from, from.off(b, 0, h), c0), y = *rotary::chunk_at(from, from.off(b, 0, h), c1);
    if (turns) {
      float2 cs[8];
      for (int e = 0; e < 8; ++e) cs[e] = rotary::cos_sin(p.rot, p.rot.inv_freq[8 * i + e], position);
      rotary::turn<T>(x, y, cs, p.rot.interleaved != 0);
    }
    *rotary::chunk_at(to, to.off(b, 0, h), c0) = x;
    *rotary::chunk_at(to, to.off(b, 0, h), c1) = y;
  }
}

// Copies a tile's rows one by one: where a page ends in it, where a page is missing, and where the token's own row is.  Lane l finds the K row
// (l < 16) or the V row of key l % 16; page0 and page1: the pages of the tile's first and last row.
template <int D>
__device__ __forceinline__ void mixed_tile(const DecodeParams& p, const Walk& w, int tile, int h, int page0, int page1, uint32_t slot, uint2* mask) {
  constexpr int kChunks = D / 8, kRows = 32 / kChunks, kCopies = kTile / kRows;
  const Sequence& s = w.s;
  const int lane = threadIdx.x & 31, r = lane / kChunks, c = lane % kChunks;
  const bool of_v = lane >= 16;
  const unsigned char* row = static_cast<const unsigned char*>(p.pages.k.ptr);
  int page = -1;
  bool valid, own = false;           // seen; the token's own, which is copied also where it has no page
  if (tile < s.cached_tiles) {
    const int key = tile * kTile + (lane & 15);
    valid = key < s.len;
    own = valid && key >= s.held;
    if (valid) {
      const int which = (int)p.pages.by_page.div((uint32_t)key);
      if (p.pages.page_size < kTile) page = __ldg(p.pages.table + w.b * p.pages.table_stride + which);      // a tile may lie in more than two
      else page = which == (int)p.pages.by_page.div((uint32_t)(tile * kTile)) ? page0 : page1;
      const int slot_of = key - which * p.pages.page_size;
      valid = page >= 0 && page < p.pages.num_pages;
      if (!valid) {
        wrong(kBadPage);
        page = -1;
      }
      if (own) row = of_v ? static_cast<const unsigned char*>(p.v.ptr) + 2 * p.v.off(w.b, 0, h) : static_cast<const unsigned char*>(p.k.ptr) + 2 * p.k.off(w.b, 0, h);
      else if (valid) row = of_v ? static_cast<const unsigned char*>(p.pages.v.ptr) + 2 * p.pages.v.off(page, slot_of, h) : row + 2 * p.pages.k.off(page, slot_of, h);
    }
  } else {
    const int d = (tile - s.cached_tiles) * kTile + (lane & 15), pos = (int)p.by_L.div((uint32_t)d), layer = d - pos * p.L;
    valid = d < s.depth;
    if (valid) row = of_v ? static_cast<const unsigned char*>(p.vd.ptr) + 2 * (p.vd.off(w.b, layer, h) + pos * p.vd_sp)
                          : static_cast<const unsigned char*>(p.kd.ptr) + 2 * (p.kd.off(w.b, layer, h) + pos * p.kd_sp);
  }
  const uint32_t seen = __ballot_sync(0xffffffffu, valid) & 0xffffu, its_own = __ballot_sync(0xffffffffu, own) & 0xffffu, there = seen | its_own;
  if (its_own == 0 ? lane == 0 : lane == __ffs(its_own) - 1) *mask = make_uint2(seen | (uint32_t)__ffs(its_own) << 16, page);
  const unsigned long long at = reinterpret_cast<unsigned long long>(row);
#pragma unroll 2
  for (int i = 0; i < kCopies; ++i) {
    const int n = i * kRows + r;
    const bool ok = (there >> n) & 1u;
    const unsigned long long k = __shfl_sync(0xffffffffu, at, n) + c * 16, v = __shfl_sync(0xffffffffu, at, 16 + n) + c * 16;
    copy16(slot + n * D * 2 + ((c ^ k_swizzle(n)) << 4), reinterpret_cast<const void*>(k), ok);
    copy16(slot + (kTile + n) * D * 2 + ((c ^ (n & 7)) << 4), reinterpret_cast<const void*>(v), ok);
  }
}

// A tile's K (or V) rows, each `stride` elements behind the one before; from row `count` on zeros.  `from`: this lane's chunk of row `row`, which
// is the first copy's and goes to `to`.  The rows of copy i swizzle as those of the first do, but for bits that are known of i.
template <int D, bool kV> __device__ __forceinline__ void copy_rows(uint32_t to, const void* from, int64_t stride, int row, int count) {
  constexpr int kRows = 32 / (D / 8), kCopies = kTile / kRows;
  const unsigned char* at = static_cast<const unsigned char*>(from);
#pragma unroll
  for (int i = 0; i < kCopies; ++i, at += kRows * 2 * stride)
    copy16((to ^ ((kV ? i * kRows & 7 : k_swizzle(i * kRows & 7)) << 4)) + i * kRows * D * 2, at, row + i * kRows < count);
}

// Copies the tiles of one warp, ahead of their use.
template <int D> struct Loader {
  Walk w;
  int tile;                          // this warp's next one, of w
  int team, rank;                    // the team's size, this warp's place in it
  int base, page0, page1;            // pages of the first and the last key of this lane's tile, base + team lane, fetched ahead for 32 of them
  bool more;
  uint32_t ring;
  int stage;
  uint32_t to_k, to_v;               // where this lane's chunk of the first copy goes in a stage

  static constexpr int kChunks = D / 8;

  // A unit's part is walked from its end: the token's own row comes first, and what is written for it is on its way before the rest.
  __device__ __forceinline__ int from_end(int n) const { return w.t0 + w.t1 - 1 - n; }
  __device__ __forceinline__ void settle(const DecodeParams& p, int units, bool fetch) {      // at a tile of this warp, or at the end
    while (more && tile >= w.t1) {
      more = w.next(p, units);
      tile = w.t0 + rank;
      fetch = true;
    }
    if (!(fetch || tile == base + 32 * team)) return;
    base = tile;
    page0 = page1 = -1;
    const int mine = tile + team * (int)(threadIdx.x & 31);
    if (!more || mine >= w.t1 || from_end(mine) >= w.s.cached_tiles) return;
    const int first = from_end(mine) * kTile;
    const int* row = p.pages.table + w.b * p.pages.table_stride;
    page0 = __ldg(row + p.pages.by_page.div((uint32_t)first));
    page1 = __ldg(row + p.pages.by_page.div((uint32_t)min(first + kTile, w.s.len) - 1u));
  }
  __device__ __forceinline__ void start(const DecodeParams& p, int units, int team_, int rank_, const Walk& from, uint32_t ring_) {
    w = from; more = true; team = team_; rank = rank_; tile = w.t0 + rank; stage = 0; ring = ring_;
    const int lane = threadIdx.x & 31, r = lane / kChunks, c = lane % kChunks;
    to_k = r * D * 2 + (c ^ k_swizzle(r)) * 16;
    to_v = kTile * D * 2 + r * D * 2 + (c ^ r) * 16;
    settle(p, units, true);
  }
  // Issues the copies of one tile (none at the end); `masks` in shared memory get a bit for each key that is there, and from bit 16 on
  // the number, from 1, of the token's own, with its page.
  __device__ __forceinline__ void issue(const DecodeParams& p, int units, int query_blocks, uint2* masks) {
    if (more) {
      const int lane = threadIdx.x & 31, r = lane / kChunks, c = lane % kChunks;
      const int h = query_blocks == 1 ? w.unit : w.unit / query_blocks, of = team == 1 ? tile - base : (tile - base) / kWarps;
      const uint32_t slot = ring + stage * stage_bytes<D>();
      const int page = __shfl_sync(0xffffffffu, page0, of), at = from_end(tile);
      // rows that follow one another in memory: of one page, or depth rows of one position
      View k = p.pages.k, v = p.pages.v;
      int64_t of_k, of_v;
      int count;
      bool run;
      if (at < w.s.cached_tiles) {
        const int first = at * kTile, row0 = first - (int)p.pages.by_page.div((uint32_t)first) * p.pages.page_size;
        count = min(w.s.len - first, kTile);
        run = first + count <= w.s.held && row0 + count <= p.pages.page_size && page >= 0 && page < p.pages.num_pages;
        of_k = k.off(page, row0 + r, h);
        of_v = v.off(page, row0 + r, h);
      } else {
        const int first = (at - w.s.cached_tiles) * kTile, pos = (int)p.by_L.div((uint32_t)first), layer = first - pos * p.L;
        count = min(w.s.depth - first, kTile);
        run = layer + count <= p.L;
        k = p.kd; v = p.vd;
        of_k = k.off(w.b, layer + r, h) + pos * p.kd_sp;
        of_v = v.off(w.b, layer + r, h) + pos * p.vd_sp;
      }
      if (__builtin_expect(run, 1)) {
        if (lane == 0) masks[stage].x = (1u << count) - 1;
        copy_rows<D, false>(slot + to_k, rotary::chunk_at(k, of_k, c), k.st, r, count);
        copy_rows<D, true>(slot + to_v, rotary::chunk_at(v, of_v, c), v.st, r, count);
      } else {
        mixed_tile<D>(p, w, at, h, page, __shfl_sync(0xffffffffu, page1, of), slot, masks + stage);
      }
      tile += team;
      settle(p, units, false);
    }
    copies_commit();
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
};

// Joins the parts that the CTAs of a cluster hold in their shared memory: rows of D at `acc`, maxima and sums at `ml`.  Each CTA
// takes every C-th group of four elements.
template <typename T, int D>
__device__ __forceinline__ void join_cluster(const DecodeParams& p, const Walk& w, int h, int q0, uint32_t acc, uint32_t ml) {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  uint32_t rank;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  for (int i = threadIdx.x * p.cluster + rank; i < kQ * D / 4; i += kThreads * p.cluster) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    if (q0 + r >= p.G) break;
    float top = -INFINITY, sum = 0.f;
    float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = 0; c0 < p.cluster; c0 += 8) {      // eight CTAs' parts on the way together
      float2 x[8];
      float4 y[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        x[c] = make_float2(-INFINITY, 0.f);
        y[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c0 + c >= p.cluster) continue;
        uint32_t at;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(ml + r * 8), "r"(c0 + c));
        asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(x[c].x), "=f"(x[c].y) : "r"(at) : "memory");
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(acc + (r * D + d) * 4), "r"(c0 + c));
        asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(y[c].x), "=f"(y[c].y), "=f"(y[c].z), "=f"(y[c].w) : "r"(at) : "memory");
      }
      float now = top;
#pragma unroll
      for (int c = 0; c < 8; ++c) now = fmaxf(now, x[c].x);
      const float base = now == -INFINITY ? 0.f : now, was = fast_exp2(top - base);
      sum *= was;
      out = make_float4(out.x * was, out.y * was, out.z * was, out.w * was);
      top = now;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float weight = fast_exp2(x[c].x - base);
        sum = fmaf(x[c].y, weight, sum);
        out = make_float4(fmaf(y[c].x, weight, out.x), fmaf(y[c].y, weight, out.y), fmaf(y[c].z, weight, out.z), fmaf(y[c].w, weight, out.w));
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint2* to = reinterpret_cast<uint2*>(static_cast<unsigned char*>(p.o.ptr) + 2 * (p.o.off(w.b, q0 + r, h) + d));
    *to = make_uint2(Pack<T>::pack(out.x * inv, out.y * inv), Pack<T>::pack(out.z * inv, out.w * inv));
    if (d == 0) p.lse[((int64_t)w.b * p.G + q0 + r) * p.H + h] = top + log2f(sum);
  }
  // Nobody leaves while it is read.  What has been read has been used above; nothing else is waited for (a release would wait for o's stores).
  asm volatile("barrier.cluster.arrive.relaxed;\n\tbarrier.cluster.wait;" ::: "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<D>()) decode_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint2 s_masks[kWarps][kStages];
  __shared__ float2 s_ml[kWarps][kQ];
  __shared__ float2 s_cs[D / 2];
  __shared__ float2 s_part_ml[kQ];
  __shared__ Range s_range;                  // read at units' ends alone: not worth registers
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane >> 2, t = lane & 3;
  const int query_blocks = (p.G + kQ - 1) / kQ, units = p.H * query_blocks;
  const uint32_t ring = smem_u32(smem) + warp * kStages * stage_bytes<D>();
  float* s_acc = reinterpret_cast<float*>(smem + (size_t)kWarps * kStages * stage_bytes<D>());

  grid_before();
  grid_started();
  Walk w;
  int64_t at = 0;                            // the place of the walk's unit in the row of all units
  int team = kWarps;
  if (p.cluster > 0) {
    locate_cluster(p, units, w);
  } else if (p.cluster == kByWarps) {
    team = 1;
    if (!locate_units(p, units, w)) return;
  } else {
    Range range;
    const bool work = locate(p, units, reinterpret_cast<int*>(s_acc), team, range, w, at);
    if (lane == 0) s_range = range;          // the same from all warps, and read by the one that has written it
    __syncwarp();
    if (!work) {
      if (lane == 0 && (team == 1 || warp == 0)) p.parts[warp * gridDim.x + blockIdx.x] = make_int2(0, team == 1 ? -1 : 0);
      return;
    }
  }
  const int rank = team == 1 ? 0 : warp;
  const uint32_t worker = team == 1 ? blockIdx.x * kWarps + warp : blockIdx.x;
  Loader<D> loader;
  loader.start(p, units, team, rank, w, ring);

  // places of this lane's chunks in a stage: K of row g (even and odd j), V of row lane % 16, chunk lane / 16
  const uint32_t k_even = g * D * 2 + (t ^ k_swizzle(g)) * 16, k_odd = g * D * 2 + ((4 + t) ^ k_swizzle(g)) * 16;
  const uint32_t v_place = (kTile + lane % 16) * D * 2 + ((lane >> 4) ^ (lane & 7)) * 16;
  int stage = 0, turned_b = -1, tile = 0, h = 0, q0 = 0;
  uint32_t qh[D / 32][4], ql[D / 32][4];     // this lane's part of the queries, in two 16-bit halves
  float m = 0.f, l = 0.f, acc[D / 8][4];
  float2* cs = team == 1 ? reinterpret_cast<float2*>(s_acc) + (1 + warp) * 64 : s_cs;      // behind what locate() may still be reading
  const int cs_first = team == 1 ? lane : tid;
  const double inv_freq = p.rot.inv_freq != nullptr && cs_first < p.rot.rot / 2 ? p.rot.inv_freq[cs_first] : 0.;
  // What a unit begins with: its queries' rows.
  auto fetch = [&]() {
    h = query_blocks == 1 ? w.unit : w.unit / query_blocks;
    q0 = (w.unit - h * query_blocks) * kQ;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (q0 + g < p.G) x = *rotary::chunk_at(p.q, p.q.off(w.b, q0 + g, h), 4 * j + t);
#pragma unroll
      for (int e = 0; e < 4; ++e) qh[j][e] = (&x.x)[e];
    }
  };
  // Steps 1 - kStages to -1 only copy.  A step's copies are issued between the scores' products and what waits for them, and at
  // one place, for the sake of the code's size: warps are few, and wait for instructions where a step has more of them.  For
  // the same reason what is rare is marked so (64 sequences of up to 4096 rows: 63.5 us without, 62.2 with).
  fetch();
  for (int step = 1 - kStages;; ++step) {
    float s[2][4], s2[2][4];                 // two sums each: the products of one wait for one another
    uint32_t mask = 0, slot = 0;
    if (step >= 0) {
      bool begins = step == 0;
      while (__builtin_expect(begins || tile >= w.t1, 0)) {
        if (!begins) {
          const bool row_there = q0 + g < p.G;
          // the warps' parts
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          const bool from_start = w.t0 == 0, to_end = w.t1 == w.s.tiles;
          const bool whole = p.cluster > 0 ? p.cluster == 1 : from_start && to_end;      // the same in all CTAs of a cluster, which meet below
          if (team == 1) {
            if (row_there) {
              const float inv = l == 0.f ? 0.f : 1.f / l;
              const int64_t at_row = ((int64_t)worker * 2 + (from_start ? 1 : 0)) * p.rows + g;
              uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(p.o.ptr) + 2 * (p.o.off(w.b, q0 + g, h) + 2 * t));
#pragma unroll
              for (int n = 0; n < D / 8; ++n) {      // elements 8 n + 2 t and the next
                const float x = both(acc[n][0], acc[n][2]), y = both(acc[n][1], acc[n][3]);
                if (whole) to[4 * n] = Pack<T>::pack(x * inv, y * inv);
                else *reinterpret_cast<float2*>(p.acc + at_row * D + 8 * n + 2 * t) = make_float2(x, y);
              }
              if (t == 0) {
                if (whole) p.lse[((int64_t)w.b * p.G + q0 + g) * p.H + h] = m + log2f(l);
                else p.ml[at_row] = make_float2(m, l);
              }
            }
          } else {
            __syncthreads();                         // the part before has been read
            if (t == 0) s_ml[warp][g] = make_float2(m, l);
            if (row_there) {
#pragma unroll
              for (int n = 0; n < D / 8; ++n) {      // elements 8 n + 2 t and the next
                float* to = reinterpret_cast<float*>(part_at<D>(s_acc, warp, g, 2 * n + (t >> 1))) + (t & 1) * 2;
                *reinterpret_cast<float2*>(to) = make_float2(both(acc[n][0], acc[n][2]), both(acc[n][1], acc[n][3]));
              }
            }
            __syncthreads();
            constexpr int kEach = D / 16;            // elements of a thread: 16 threads a row
            const int r = tid / 16, d0 = (tid % 16) * kEach;
            if (q0 + r < p.G) {
              float top = -INFINITY;
#pragma unroll
              for (int i = 0; i < kWarps; ++i) top = fmaxf(top, s_ml[i][r].x);
              const float base = top == -INFINITY ? 0.f : top;
              float sum = 0.f, out[kEach] = {};
#pragma unroll
              for (int i = 0; i < kWarps; ++i) {
                const float weight = fast_exp2(s_ml[i][r].x - base);
                sum = fmaf(s_ml[i][r].y, weight, sum);
#pragma unroll
                for (int e = 0; e < kEach; e += 4) {
                  const float4 x = *part_at<D>(s_acc, i, r, (d0 + e) / 4);
                  out[e] = fmaf(x.x, weight, out[e]);
                  out[e + 1] = fmaf(x.y, weight, out[e + 1]);
                  out[e + 2] = fmaf(x.z, weight, out[e + 2]);
                  out[e + 3] = fmaf(x.w, weight, out[e + 3]);
                }
              }
              if (whole) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                uint32_t packed[kEach / 2];
#pragma unroll
                for (int e = 0; e < kEach / 2; ++e) packed[e] = Pack<T>::pack(out[2 * e] * inv, out[2 * e + 1] * inv);
                uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(p.o.ptr) + 2 * (p.o.off(w.b, q0 + r, h) + d0));
#pragma unroll
                for (int e = 0; e < kEach / 2; ++e) to[e] = packed[e];
                if (d0 == 0) p.lse[((int64_t)w.b * p.G + q0 + r) * p.H + h] = top + log2f(sum);
              } else {                               // into scratch; a cluster's parts into each CTA's shared memory (its slots are free)
                const int64_t at_row = p.cluster > 0 ? r : ((int64_t)worker * 2 + (from_start ? 1 : 0)) * p.rows + r;
                float* to = (p.cluster > 0 ? reinterpret_cast<float*>(smem) : p.acc) + at_row * D + d0;
#pragma unroll
                for (int e = 0; e < kEach; ++e) to[e] = out[e];
                if (d0 == 0) (p.cluster > 0 ? s_part_ml : p.ml)[at_row] = make_float2(top, sum);
              }
            }
          }
          if (p.cluster > 0) {
            if (!whole) join_cluster<T, D>(p, w, h, q0, smem_u32(smem), smem_u32(s_part_ml));
            return;
          }
          int2* const mine = p.parts + (team == 1 ? warp * gridDim.x : 0) + blockIdx.x;
          if (!to_end) {                           // the last one of the range; begun here: how many teams hold a part of it
            if (lane == 0 && rank == 0) {
              int2 part = make_int2(0, team == 1 ? -1 : 0);
              if (from_start) {
                const Range range = s_range;
                const int64_t last = at + w.places() - 1;
                uint32_t n = (uint32_t)quotient(last - at, (uint32_t)min(range.each, (int64_t)0x7fffffff));      // the ranges are `each` long, or one more
                while (n > 0 && range.begin(worker + n) > last) --n;
                while (worker + n + 1 < range.n && range.begin(worker + n + 1) <= last) ++n;
                part = make_int2(w.b * units + w.unit, ((int)n + 1) * (team == 1 ? -1 : 1));
              }
              *mine = part;
            }
            return;
          }
          at += w.places();
          if (!w.next(p, units)) {
            if (p.cluster == 0 && lane == 0 && rank == 0) *mine = make_int2(0, team == 1 ? -1 : 0);
            return;
          }
          fetch();
        }
        const bool row_there = q0 + g < p.G;
        if (p.rot.inv_freq != nullptr) {     // one cosine and sine a thread, while the first copies are on the way
          if (turned_b != w.b)               // those of the unit before have been read: its parts have been joined
            for (int i = cs_first; i < p.rot.rot / 2; i += 32 * team)
              cs[i] = rotary::cos_sin(p.rot, i == cs_first ? inv_freq : p.rot.inv_freq[i], p.k.ptr != nullptr ? w.s.held : w.s.held - 1);
          turned_b = w.b;
          if (team == 1) __syncwarp();
          else __syncthreads();
        }
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const int chunk = 4 * j + t;
          const int64_t row = p.q.off(w.b, q0 + g, h);
#pragma unroll
          for (int e = 0; e < 4; ++e) ql[j][e] = 0;
          if (p.rot.inv_freq != nullptr && row_there && chunk * 8 < p.rot.rot) {
            float y[8];
            if (p.rot.interleaved) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 a = Pack<T>::unpack(qh[j][e]), turn = cs[chunk * 4 + e];
                y[2 * e] = fmaf(a.x, turn.x, -a.y * turn.y);
                y[2 * e + 1] = fmaf(a.y, turn.x, a.x * turn.y);
              }
            } else {
              const int half = p.rot.rot >> 4;                     // chunks
              const bool second = chunk >= half;
              const uint4 other = *rotary::chunk_at(p.q, row, second ? chunk - half : chunk + half);
              const int pair = (second ? chunk - half : chunk) * 8;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 a = Pack<T>::unpack(qh[j][e]), b = Pack<T>::unpack((&other.x)[e]);
                const float2 c0 = cs[pair + 2 * e], c1 = cs[pair + 2 * e + 1];
                y[2 * e] = fmaf(a.x, c0.x, second ? b.x * c0.y : -b.x * c0.y);
                y[2 * e + 1] = fmaf(a.y, c1.x, second ? b.y * c1.y : -b.y * c1.y);
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) split<T>(y[2 * e], y[2 * e + 1], qh[j][e], ql[j][e]);
          }
        }
        // the part that ends the unit has its last tile, which may not be empty: there is one such part
        if (__builtin_expect(p.copy_all != 0 && w.s.len == w.s.held && w.t1 == w.s.tiles && w.t0 < w.t1 && q0 == 0 && rank == 0 && lane == 0, 0))
          copy_own_row<T, D>(p, w.b, h, w.s.held);
        m = -INFINITY; l = 0.f;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        tile = w.t0 + rank;
        begins = false;
      }
      copies_wait<kStages - 2>();
      __syncwarp();                          // the other lanes' copies, and the mask; and all lanes have read the tile before
      mask = s_masks[warp][stage].x;
      slot = ring + stage * stage_bytes<D>();
      if (__builtin_expect(mask >> 16, 0)) {
        own_row<T, D>(p, w, h, (int)s_masks[warp][stage].y, q0 == 0, slot, (int)(mask >> 16) - 1, cs);
        mask &= 0xffffu;
      }
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = s2[nt][0] = s2[nt][1] = s2[nt][2] = s2[nt][3] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint4 k = lds128(slot + (j & 1 ? k_odd : k_even) + nt * 8 * D * 2 + (j >> 1) * 128);
          mma<T>(s[nt], qh[j][0], ql[j][0], qh[j][1], ql[j][1], k.x, k.y);
          mma<T>(s2[nt], qh[j][2], ql[j][2], qh[j][3], ql[j][3], k.z, k.w);
        }
      }
    }
    loader.issue(p, units, query_blocks, s_masks[warp]);
    if (step < 0) continue;
    float x[4];                            // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int nt = i >> 1, e = i & 1;
      x[i] = both(s[nt][e] + s2[nt][e], s[nt][2 + e] + s2[nt][2 + e]) * p.scale_log2;
    }
    if (mask != 0xffffu) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!((mask >> (2 * t + (i & 1) + (i >> 1) * 8)) & 1u)) x[i] = -INFINITY;
    }
    float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    top = fmaxf(top - Lift<T>::value, m);
    const float base = top == -INFINITY ? 0.f : top;
    if (__any_sync(0xffffffffu, top > m)) {
      const float shrink = fast_exp2(m - base);
      l *= shrink;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) { acc[n][0] *= shrink; acc[n][1] *= shrink; acc[n][2] *= shrink; acc[n][3] *= shrink; }
      m = top;
    }
    float pr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { pr[i] = fast_exp2(x[i] - base); l += pr[i]; }
    uint32_t ph[2], pl[2];
    split<T>(pr[0], pr[1], ph[0], pl[0]);
    split<T>(pr[2], pr[3], ph[1], pl[1]);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {      // keys 0 .. 7 and 8 .. 15 of elements 16 j .. + 7, and of 16 j + 8 .. + 15
      uint32_t v[4];
      load_transposed(v, ((slot + v_place) ^ ((j & 3) << 5)) + (j >> 2) * 128);
      mma<T>(acc[2 * j], ph[0], pl[0], ph[1], pl[1], v[0], v[1]);
      mma<T>(acc[2 * j + 1], ph[0], pl[0], ph[1], pl[1], v[2], v[3]);
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
    tile += team;
  }
}
// Joins the parts of the units that several CTAs hold.  Grid: (CTA in which the unit begins, query row).  A warp takes every eighth
// part, five of them on the way together: 40 parts, what one sequence with 8 heads has, take one trip to memory.  (One head of
// one sequence has up to 296, D = 128: eight trips.)
constexpr int kJoinWarps = 8, kJoinAhead = 5;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32, 5) join_kernel(const __grid_constant__ DecodeParams p) {
  __shared__ float s_acc[kJoinWarps][D];
  __shared__ float2 s_ml[kJoinWarps];
  grid_before();
  int2 part = p.parts[blockIdx.x];
  if (part.y == 0) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = blockIdx.y;
  const bool by_warps = part.y < 0;          // four teams' parts; or the CTA's
#pragma unroll 1
  for (int k = 0; k < (by_warps ? kWarps : 1); ++k) {
    if (k > 0) part = p.parts[k * gridDim.x + blockIdx.x];
    const int id = part.x, n = abs(part.y);
    if (n < 2) continue;                     // the same for all threads, as is what follows
    const int query_blocks = (p.G + kQ - 1) / kQ, units = p.H * query_blocks;
    const int b = id / units, u = id - b * units, h = u / query_blocks, row = (u - h * query_blocks) * kQ + r;
    if (row >= p.G) continue;
    const int64_t first = by_warps ? blockIdx.x * kWarps + k : blockIdx.x;      // the team
    auto place = [&](int i) { return ((first + i) * 2 + (i == 0 ? 1 : 0)) * p.rows + r; };
    constexpr int kEach = D / 32;
    float top = -INFINITY, sum = 0.f, out[kEach] = {};
    for (int i0 = warp; i0 < n; i0 += kJoinAhead * kJoinWarps) {
      float2 ml[kJoinAhead];
      float x[kJoinAhead][kEach];
#pragma unroll
      for (int i = 0; i < kJoinAhead; ++i) {
        const int64_t at = place(min(i0 + i * kJoinWarps, n - 1));      // beyond the last one: it again, unused
        ml[i] = p.ml[at];
        const float* from = p.acc + at * D + lane * kEach;
        if constexpr (kEach == 4) *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(from);
        else *reinterpret_cast<float2*>(x[i]) = *reinterpret_cast<const float2*>(from);
      }
#pragma unroll
      for (int i = 0; i < kJoinAhead; ++i) {
        if (i0 + i * kJoinWarps >= n) break;
        const float now = fmaxf(top, ml[i].x), base = now == -INFINITY ? 0.f : now, was = fast_exp2(top - base), is = fast_exp2(ml[i].x - base);
        sum = sum * was + ml[i].y * is;
#pragma unroll
        for (int e = 0; e < kEach; ++e) out[e] = out[e] * was + x[i][e] * is;
        top = now;
      }
    }
    __syncthreads();                         // the unit before has been read
#pragma unroll
    for (int e = 0; e < kEach; ++e) s_acc[warp][lane * kEach + e] = out[e];
    if (lane == 0) s_ml[warp] = make_float2(top, sum);
    __syncthreads();
    if (threadIdx.x >= D / 2) continue;      // two elements a thread
    const int held_by = min(n, kJoinWarps), d = threadIdx.x;
    for (int i = 0; i < held_by; ++i) top = fmaxf(top, s_ml[i].x);
    const float base = top == -INFINITY ? 0.f : top;
    float x = 0.f, y = 0.f;
    sum = 0.f;
    for (int i = 0; i < held_by; ++i) {
      const float weight = fast_exp2(s_ml[i].x - base);
      sum = fmaf(s_ml[i].y, weight, sum);
      x = fmaf(s_acc[i][2 * d], weight, x);
      y = fmaf(s_acc[i][2 * d + 1], weight, y);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(p.o.ptr) + 2 * p.o.off(b, row, h))[d] = Pack<T>::pack(x * inv, y * inv);
    if (d == 0) p.lse[((int64_t)b * p.G + row) * p.H + h] = top + log2f(sum);
  }
}

}  // namespace paged
}  // namespace moda
