// Rotary positions, and the paged KV cache's append with the rotation on the way.
//
// A pair (x1, x2) of a vector at position p is turned by the angle a = p f of its frequency f (radians a
// position): y1 = s (x1 cos a - x2 sin a), y2 = s (x2 cos a + x1 sin a).  The gradient goes the other way
// round, by -a.  Pairs are elements (i, i + rot / 2) ("half") or (2 i, 2 i + 1) ("interleaved") of the first
// rot elements of a head; the others pass through.
//
// The angle is reduced in whole turns and in integers: f / 2 pi modulo 1 as a 64-bit fraction (from a product in two
// parts), times p with the product's overflow dropped, is p f / 2 pi modulo 1, since what overflows are whole turns.  A position of
// 2^31 leaves 2^-32 of a turn of error, where an angle in 32-bit floating point is off by whole radians.
//
// The operators move bytes: x is read and y written once.  A warp takes a token: every vector of
// the token (G H query heads and H key heads) turns by the same angles, so a lane computes its share of the
// sines once, fetches the others with shuffles, and walks the vectors with two 16-byte chunks each that hold
// eight pairs.  The first rows are on the way while the sines (and a page) are looked up, and what a lane has under way is
// kept small enough for 32 warps an SM: 65536 tokens of 40 heads of 128 take 202 us (6.6 TB/s), against 218 with four
// vectors a lane and 20 warps, and 239 with two vectors and as many registers as the compiler would take.
#pragma once
#include "common.cuh"

namespace moda {
namespace rotary {

// Division of a number below 2^31 by a fixed one, 2^s < d <= 2^(s+1).  m = ceil(2^(32+s) / d) fits 32 bits, and
// n m / 2^(32+s) exceeds n / d by less than n / 2^(32+s) < 2^-(s+1) <= 1 / d: too little to reach the next whole number.
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() : d(1), m(0), s(0) {}
  explicit FastDiv(uint32_t div) : d(div), m(0), s(0) {
    if (div <= 1) return;
    while ((2ull << s) < div) ++s;
    m = (uint32_t)(((1ull << (32 + s)) + div - 1) / div);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, m) >> s; }
};

struct Args {                // how vectors are turned
  const double* inv_freq;    // rot / 2 frequencies, radians a position; nullptr: not at all
  int rot;                   // elements of a head that turn: a multiple of 16
  int interleaved;
  int inverse;               // by the negative angle
  float scale;
};

// Cosine and sine of position pos at frequency f, times the factor.  Whole quarter turns are taken off in integers; what is left, at
// most an eighth of a turn, becomes a number of 53 bits of its own (a slow pair's angle near the start is a small part of a turn: the
// upper 32 bits of the fraction alone would hold 1.6e-8 radians, of base 1e7 stretched by 8, with an error of a tenth), x = pi / 4 at most,
// which goes through the Taylor series in 64 bits (first terms left out: x^13 / 13! = 7e-12, x^12 / 12! = 1.2e-10), so that the
// error that counts is the rounding to 32 bits at the end.  A lane does this once or twice a token.
__device__ __forceinline__ float2 cos_sin(const Args& a, double f, long long pos) {
  constexpr double kHi = 0.15915494309189535, kLo = -9.839338337591243e-18;      // 1 / 2 pi
  const double all = f * kHi, rest = fma(f, kLo, fma(f, kHi, -all));
  const unsigned long long step = (unsigned long long)((all - floor(all)) * 18446744073709551616.0) + (unsigned long long)(long long)(rest * 18446744073709551616.0);
  const unsigned long long turn = step * (unsigned long long)pos;                  // of a turn, times 2^64
  const unsigned long long quarters = (turn + (1ull << 61)) >> 62;
  const double x = (double)(long long)(turn - (quarters << 62)) * 3.4061215800865545e-19, x2 = x * x;      // 2 pi / 2^64
  double s = -1. / 39916800., c = -1. / 3628800.;
  s = fma(s, x2, 1. / 362880.);
  c = fma(c, x2, 1. / 40320.);
  s = fma(s, x2, -1. / 5040.);
  c = fma(c, x2, -1. / 720.);
  s = fma(s, x2, 1. / 120.);
  c = fma(c, x2, 1. / 24.);
  s = fma(s, x2, -1. / 6.);
  c = fma(c, x2, -1. / 2.);
  s = fma(s * x2, x, x) * (double)a.scale;
  c = fma(c, x2, 1.) * (double)a.scale;
  float fs = (float)s, fc = (float)c;
  if (quarters & 1) { const float t = fc; fc = -fs; fs = t; }
  if (quarters & 2) { fc = -fc; fs = -fs; }
  return make_float2(fc, a.inverse ? -fs : fs);
}

// The two chunks (of 8 elements) of lane item c < D / 16, and whether they turn.  Item c holds pairs 8 c .. 8 c + 7.
__device__ __forceinline__ bool item_chunks(const Args& a, int c, int& c0, int& c1) {
  const int turning = a.rot >> 4;
  if (c < turning && !a.interleaved) { c0 = c; c1 = c + turning; return true; }
  c0 = 2 * c; c1 = 2 * c + 1;
  return c < turning;
}

// Turns the eight pairs of two chunks.  cs[i]: cosine and sine of pair i.
template <typename T> __device__ __forceinline__ void turn(uint4& x, uint4& y, const float2 (&cs)[8], bool interleaved) {
  uint32_t* xs = &x.x;
  uint32_t* ys = &y.x;
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = Pack<T>::unpack(xs[i]), b = Pack<T>::unpack(ys[i]);
      const float2 p = cs[i], q = cs[4 + i];
      xs[i] = Pack<T>::pack(fmaf(a.x, p.x, -a.y * p.y), fmaf(a.y, p.x, a.x * p.y));
      ys[i] = Pack<T>::pack(fmaf(b.x, q.x, -b.y * q.y), fmaf(b.y, q.x, b.x * q.y));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = Pack<T>::unpack(xs[i]), b = Pack<T>::unpack(ys[i]);
      const float2 p = cs[2 * i], q = cs[2 * i + 1];
      xs[i] = Pack<T>::pack(fmaf(a.x, p.x, -b.x * p.y), fmaf(a.y, q.x, -b.y * q.y));
      ys[i] = Pack<T>::pack(fmaf(b.x, p.x, a.x * p.y), fmaf(b.y, q.x, a.y * q.y));
    }
  }
}

// The eight cosines and sines of this lane's item at its token's position pos.  Of the warp's 32 lanes, 32 / (C kTokens) have the same item
// and token and compute an equal share each.
template <int C, int kTokens = 1> __device__ __forceinline__ void item_cos_sin(const Args& a, int lane, long long pos, float2 (&cs)[8]) {
  constexpr int kShare = 32 / (C * kTokens), kEach = 8 / kShare;
  const int c = lane % C, v = lane / C % kShare;
  float2 mine[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    mine[i] = c < (a.rot >> 4) ? cos_sin(a, a.inv_freq[8 * c + v * kEach + i], pos) : make_float2(1.f, 0.f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int from = lane + (i / kEach - v) * C;
    cs[i].x = __shfl_sync(0xffffffffu, mine[i % kEach].x, from);
    cs[i].y = __shfl_sync(0xffffffffu, mine[i % kEach].y, from);
  }
}

__device__ __forceinline__ uint4* chunk_at(const View& x, int64_t off, int chunk) {
  return reinterpret_cast<uint4*>(static_cast<unsigned char*>(x.ptr) + 2 * (off + chunk * 8));
}

// Positions of the tokens: a tensor of 32- or 64-bit whole numbers, or their index plus an offset.
struct Positions {
  const void* data;
  int64_t sb, st, offset;
  int is64;
  __device__ __forceinline__ long long at(int b, int t) const {
    if (data == nullptr) return offset + t;
    const int64_t i = b * sb + t * st;
    return is64 ? static_cast<const long long*>(data)[i] : (long long)static_cast<const int*>(data)[i];
  }
};

struct RotaryParams {
  View q, k, q_out, k_out;   // q [B, T G, H, D], k [B, T, H, D] (pointers nullptr: none)
  Positions pos;
  Args rot;
  int B, T, H, G;
  int vectors, per_warp;     // a token's vectors; those that one warp takes
  FastDiv by_h, by_t;
};

constexpr int kThreads = 128, kBlocks = 8;      // an SM: 32 warps, 64 registers a thread
constexpr int kBatch = 2;    // vectors whose loads a lane has under way together

// Grid: x over the tokens (kTokens a warp), y over shares of a token's vectors.
template <typename T, int D, int kTokens>
__global__ void __launch_bounds__(kThreads, kBlocks) rotary_kernel(const __grid_constant__ RotaryParams p) {
  grid_before();
  constexpr int C = D / 16, kLanes = 32 / (C * kTokens);      // kLanes vectors of a token at a time
  const int lane = threadIdx.x % 32, c = lane % C;
  const int first = blockIdx.y * p.per_warp, last = min(first + p.per_warp, p.vectors);
  int c0, c1;
  const bool turns = item_chunks(p.rot, c, c0, c1);
  const bool interleaved = p.rot.interleaved != 0;
  const int64_t tok = ((int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32) * kTokens + lane / (C * kLanes);
  const bool active = tok < (int64_t)p.B * p.T;
  const int b = active ? (int)p.by_t.div((uint32_t)tok) : 0, t = active ? (int)(tok - (int64_t)b * p.T) : 0;
  float2 cs[8];
  for (int step = 0; first + step * kBatch * kLanes < last; ++step) {      // uniform over the warp
    const int v0 = first + step * kBatch * kLanes + lane / C % kLanes;
    uint4 x[kBatch], y[kBatch];
    int64_t out[kBatch];
    bool is_k[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int v = v0 + i * kLanes;
      if (v >= last || !active) continue;
      const int g = (int)p.by_h.div((uint32_t)v), h = v - g * p.H;
      is_k[i] = g == p.G;
      const View& in = is_k[i] ? p.k : p.q;
      const int64_t row = is_k[i] ? t : (int64_t)t * p.G + g, off = in.off(b, row, h);
      out[i] = (is_k[i] ? p.k_out : p.q_out).off(b, row, h);
      x[i] = *chunk_at(in, off, c0);
      y[i] = *chunk_at(in, off, c1);
    }
    if (step == 0) item_cos_sin<C, kTokens>(p.rot, lane, p.pos.at(b, t), cs);      // while they are on the way
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (v0 + i * kLanes >= last || !active) continue;
      if (turns) turn<T>(x[i], y[i], cs, interleaved);
      const View& to = is_k[i] ? p.k_out : p.q_out;
      *chunk_at(to, out[i], c0) = x[i];
      *chunk_at(to, out[i], c1) = y[i];
    }
  }
}

}  // namespace rotary

// ------------------------------------------------------------------ paged KV cache
namespace paged {

using rotary::FastDiv;

// Sequences of a paged cache.  Position n of sequence b lives in row n % page_size of page table[b][n / page_size].
struct Pages {
  View k, v;                 // [num_pages, page_size, H, D]
  const int* table;          // [B, max_pages]
  int64_t table_stride;
  const int* seq_lens;       // [B]
  int num_pages, page_size, max_pages;
  FastDiv by_page;
  int room;                  // positions that a row of the table covers, at most 2^31 - 1
};

// What a call found wrong in its tables or lengths: 2 << 8 | one of these, kept until the host reads it.  The
// rows concerned are left out (of the softmax, of the append); nothing outside the tensors is touched.
enum Wrong : int { kBadPage = 1, kBadLength = 2 };
__device__ int g_wrong;
__device__ __forceinline__ void wrong(int what) { atomicCAS(&g_wrong, 0, (2 << 8) | what); }

struct AppendParams {
  View k, v;                 // [B, T, H, D]
  Pages pages;
  const int* lengths;        // [B], nullptr: T tokens each
  rotary::Args rot;          // of the keys
  int B, T, H;
  int per_warp;              // of a token's 2 H vectors
  FastDiv by_t;
};

template <typename T, int D, int kTokens>
__global__ void __launch_bounds__(rotary::kThreads, rotary::kBlocks) append_kernel(const __grid_constant__ AppendParams p) {
  using namespace rotary;
  grid_before();
  constexpr int C = D / 16, kLanes = 32 / (C * kTokens);
  const int lane = threadIdx.x % 32, c = lane % C;
  const int first = blockIdx.y * p.per_warp, last = min(first + p.per_warp, 2 * p.H);
  int c0, c1;
  const bool turns = item_chunks(p.rot, c, c0, c1) && p.rot.inv_freq != nullptr;
  const bool interleaved = p.rot.interleaved != 0;
  const int64_t tok = ((int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32) * kTokens + lane / (C * kLanes);
  bool active = tok < (int64_t)p.B * p.T;
  const int b = active ? (int)p.by_t.div((uint32_t)tok) : 0, t = active ? (int)(tok - (int64_t)b * p.T) : 0;
  if (active && p.lengths != nullptr) {
    const int given = p.lengths[b];
    if (given < 0 || given > p.T) wrong(kBadLength);
    active = t < given;
  }
  if (!__any_sync(0xffffffffu, active)) return;
  float2 cs[8];
  int page = 0, slot = 0;
  for (int step = 0; first + step * kBatch * kLanes < last; ++step) {      // uniform over the warp
    const int v0 = first + step * kBatch * kLanes + lane / C % kLanes;
    uint4 x[kBatch], y[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int v = v0 + i * kLanes;
      if (v >= last || !active) continue;
      const View& in = v < p.H ? p.k : p.v;
      const int64_t off = in.off(b, t, v < p.H ? v : v - p.H);
      x[i] = *chunk_at(in, off, c0);
      y[i] = *chunk_at(in, off, c1);
    }
    if (step == 0) {                         // the place and the angles, while the rows are on the way
      const int64_t n = (int64_t)p.pages.seq_lens[b] + t;
      if (active && (n < 0 || n >= p.pages.room)) {
        active = false;
        wrong(kBadLength);
      }
      if (active) {
        const int which = (int)p.pages.by_page.div((uint32_t)n);
        page = p.pages.table[b * p.pages.table_stride + which];
        slot = (int)n - which * p.pages.page_size;
      }
      if (p.rot.inv_freq != nullptr && first < p.H) item_cos_sin<C, kTokens>(p.rot, lane, n, cs);
      if (active && (page < 0 || page >= p.pages.num_pages)) {
        active = false;
        wrong(kBadPage);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int v = v0 + i * kLanes;
      if (v >= last || !active) continue;
      if (turns && v < p.H) turn<T>(x[i], y[i], cs, interleaved);
      const View& to = v < p.H ? p.pages.k : p.pages.v;
      const int64_t off = to.off(page, slot, v < p.H ? v : v - p.H);
      *chunk_at(to, off, c0) = x[i];
      *chunk_at(to, off, c1) = y[i];
    }
  }
}

}  // namespace paged
}  // namespace moda
