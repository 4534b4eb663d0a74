// The paged 4-bit cache of keys and values: quantising rows as they are written, reading them back as values, and
// attention over the cache.
//
// Format.  A row (one token of one kv head) is cut into groups of GS = min(32, D) neighbouring elements.  A group has a
// bf16 scale s = amax / 7 (nearest even) and codes c = sign(x) floor(|x| / s + 1/2) in -7 .. 7, and stands for s c.
//   * s is at most half a bf16 step off amax / 7, so that amax / s < 7.5 and no code leaves the range.
//   * s is 0 (and with it every value) where it would be below the smallest normal number, and a NaN with its sign bit
//     set where the group holds an infinity or a NaN: all of the group then reads as NaN.
//   * |x| / s is taken as |x| (1 / s) (1 + 2^-20).  Exact halves go up either way; a quotient that is no half lies at
//     least 2^-16 of its size away from one (x has 11 significant bits, s has 8), so the nudge moves none across.
// s c is exact in fp16 (8 + 3 bits) and rounded once in bf16.
//
// Layout.  Codes are stored as nibbles c + 8, rows of D / 2 bytes, [page][kv head][token of the page][D / 2], scales
// [page][kv head][token][D / GS]: the tokens of a page and head are one piece of memory.  Within a row the elements lie
// as the matrix instructions of the attention kernel want them, so that a thread's operands are one load:
//   keys    word t NG + gi holds elements 32 gi + 8 t .. + 7 (t = 0..3: the four lanes that share a column), rotated left by 2
//   values  half-word g NG + gi holds elements 32 gi + 4 g .. + 3 (g = 0..7: the eight lanes that share a row), rotated left by 2
// (head dim 16: half-words and bytes in order, not rotated).  Rotated, the first two nibbles lie in bits 2..9 of their
// half, and after a rotation by 8 the next two do: the mantissa of a half-precision number.
#include <cuda.h>

#include <type_traits>

#include "faws_internal.cuh"
#include "faws_tc_host.cuh"
#include "faws_tc_ptx.cuh"

namespace faws {
namespace {
using namespace ptx;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
#define FAWS_NEG_INF (__int_as_float(0xff800000))
constexpr int kBadPage = 2;  // bit of the device's status word: a page or a length that the cache does not have

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (nibble - 8) * scale of both halves, rounded once; `scale` a bf16 number
template <typename T> __device__ __forceinline__ uint32_t code_times_scale(uint32_t nibbles, uint32_t scale);
template <> __device__ __forceinline__ uint32_t code_times_scale<__half>(uint32_t nibbles, uint32_t scale) {
  nibbles |= 0x64006400u;  // 1024 + n
  const __half2 c = __hsub2(*reinterpret_cast<__half2*>(&nibbles), __floats2half2_rn(1032.f, 1032.f));
  const float sf = __uint_as_float(scale << 16);
  if (scale >= 0x3780u) {  // from 2^-16 on a bf16 number is an fp16 one (of a group of fp16 numbers: at most 2^13.2), or NaN
    const __half2 v = __hmul2(c, __float2half2_rn(sf));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const float2 f = __half22float2(c);
  const __half2 v = __floats2half2_rn(f.x * sf, f.y * sf);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t code_times_scale<__nv_bfloat16>(uint32_t nibbles, uint32_t scale) {
  nibbles |= 0x43004300u;  // 128 + n
  scale |= scale << 16;
  const __nv_bfloat162 c = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&nibbles), __floats2bfloat162_rn(136.f, 136.f));
  const __nv_bfloat162 v = __hmul2(c, *reinterpret_cast<__nv_bfloat162*>(&scale));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Positions that a sequence's row of the table has room for.  Those behind them do not exist: rows are not written there and read as
// NaN, keys are NaN.
__device__ __forceinline__ int table_room(const CacheBatch& c, int page_shift) {
  const long long room = (long long)c.max_pages << page_shift;
  return room > 0x3fffffff ? 0x3fffffff : (int)room;
}
// Length of sequence b, 0 where `lengths` says less; *bad where it says less or more than `room`.
__device__ __forceinline__ int told_length(const CacheBatch& c, int room, int b, bool* bad) {
  const int n = c.lengths[b];
  if (n < 0 || n > room) *bad = true;
  return max(0, n);
}

// ---------------------------------------------------------------------------------------------- write, read
// A thread has 8 neighbouring elements of a row; TPR = D / 8 threads a row, the four (D 16: two) of a group next to each other.
// Bound by HBM: 2 bytes read and 9/16 written an element (reading back: the other way round).  A CTA takes consecutive rows
// of one sequence and head, a thread four of them, so that what a row costs beside its elements is little, or one where a
// sequence has no more than a CTA's.
struct CacheRows {
  const void* src[2];  // write: k, v; read: unused
  void* dst[2];        // read: k, v
  int64_t sb[2], sh[2], ss[2];
  int rows;            // of each sequence
  int tiles;           // CTAs that the rows of a sequence and head take
  int vec;             // 16-byte accesses to them
};
constexpr int kRowsEach = 4;

// What the rows of a CTA have in common, and where row m of its sequence and head lies in the cache's tensors (-1: on a page that
// does not exist).  The CTA's rows mostly lie on one page, which is then looked up once.
struct RowPlace {
  const int32_t* table;
  int first;           // position of row 0
  int stop;            // the rows from here on lie behind the table, or do not belong to the call
  int shift, pages, Hk, hk;
  int one;             // the page of all rows, or kSeveral
  static constexpr int kSeveral = -0x7fffffff;
  __device__ __forceinline__ bool real(int m) const { return m < stop && first + m >= 0; }
  __device__ __forceinline__ int64_t at(int m, bool* bad) const {
    const int pos = first + m, page = one != kSeveral ? one : table[pos >> shift];
    if ((unsigned)page >= (unsigned)pages) {
      *bad = true;
      return -1;
    }
    return (((int64_t)page * Hk + hk) << shift) + (pos & ((1 << shift) - 1));
  }
};
// of the CTA's rows [m0, m1)
__device__ __forceinline__ RowPlace row_place(const CacheParams& c, const CacheBatch& bt, int rows, int b, int hk, int m0, int m1,
                                              bool* bad) {
  RowPlace p;
  p.table = bt.table + (int64_t)b * bt.table_stride;
  const int room = table_room(bt, c.page_shift);
  p.first = told_length(bt, room, b, bad) - rows;
  p.stop = min(rows, room - p.first);
  p.shift = c.page_shift;
  p.pages = c.pages;
  p.Hk = c.Hk;
  p.hk = hk;
  const int lo = max(p.first + m0, 0) >> c.page_shift, hi = (p.first + min(m1, p.stop) - 1) >> c.page_shift;
  p.one = lo == hi ? p.table[lo] : RowPlace::kSeveral;  // (hi < 0, or before lo: no row is real)
  return p;
}

// The words of a row of values as they lie in memory, from the words of elements (`to` true), or back.  Word p of the row: half-words
// g NG + gi of 2 p and 2 p + 1; the word of elements w = 4 gi + t: half-words of g = 2 t and 2 t + 1, group gi.
template <int D>
__device__ __forceinline__ uint32_t exchange_halves(uint32_t word, int w, bool to) {
  if constexpr (D < 64) return word;  // one group: the same order
  else {
  constexpr int NG = D / 32, TPR = D / 8;
  const int lane0 = (threadIdx.x & 31) & ~(TPR - 1);
  // to memory: position w is g = 2 w / NG, groups gi and gi + 1, from the words 4 gi + g / 2 and 4 (gi + 1) + g / 2, half g & 1
  // from memory: word 4 gi + t takes half-words (2 t) NG + gi and (2 t + 1) NG + gi: words t NG + gi / 2 and + NG / 2, half gi & 1
  const int g = 2 * w / NG, gi = to ? 2 * w % NG : w / 4, t = w % 4;
  const int from0 = to ? 4 * gi + g / 2 : t * NG + gi / 2;
  const uint32_t a = __shfl_sync(0xffffffffu, word, lane0 + from0);
  const uint32_t b = __shfl_sync(0xffffffffu, word, lane0 + from0 + (to ? 4 : NG / 2));
  return __byte_perm(a, b, ((to ? g : gi) & 1) ? 0x7632 : 0x5410);
  }
}
// each half rotated left by 2, and right
__device__ __forceinline__ uint32_t rotate_halves(uint32_t x) { return (x << 2 & 0xfffcfffcu) | (x >> 14 & 0x00030003u); }
__device__ __forceinline__ uint32_t rotate_halves_back(uint32_t x) { return (x >> 2 & 0x3fff3fffu) | (x << 14 & 0xc000c000u); }

// A CTA's rows: `lanes` at a time from row `first` of sequence b and head hk on.
struct RowTile {
  int b, hk, first, lanes;
};

template <typename T, int D, bool VALUES, bool WHOLE, int EACH>
__device__ __forceinline__ void write_rows(const CacheParams& c, const CacheRows& r, const RowPlace& place, const RowTile& t, bool* bad) {
  constexpr int TPR = D / 8, NG = D >= 32 ? D / 32 : 1, GL = D >= 32 ? 4 : 2;
  constexpr uint32_t kInfinity = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  const int w = threadIdx.x % TPR, lanes = t.lanes, m0 = t.first + threadIdx.x / TPR;
  // WHOLE: the rows lie one behind the other
  const int64_t row0 = WHOLE ? place.at(m0, bad) : 0;
  const int64_t ss = r.ss[VALUES];
  const T* src = static_cast<const T*>(r.src[VALUES]) + t.b * r.sb[VALUES] + t.hk * r.sh[VALUES] + m0 * ss + w * 8;
  unsigned char* codes = static_cast<unsigned char*>(VALUES ? c.v_codes : c.k_codes) + (D >= 32 && !VALUES ? (w % 4) * NG + w / 4 : w) * 4;
  uint16_t* scales = static_cast<uint16_t*>(VALUES ? c.v_scales : c.k_scales) + w / GL;
  uint4 in[EACH];
#pragma unroll
  for (int y = 0; y < EACH; ++y) {
    in[y] = make_uint4(0u, 0u, 0u, 0u);
    if (WHOLE || place.real(m0 + y * lanes)) {
      const T* from = src + y * lanes * ss;
      if (WHOLE || r.vec) in[y] = *reinterpret_cast<const uint4*>(from);
      else {
        uint16_t e[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) e[x] = reinterpret_cast<const uint16_t*>(from)[x];
        in[y] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
      }
    }
  }
#pragma unroll
  for (int y = 0; y < EACH; ++y) {
    const int m = m0 + y * lanes;
    const uint32_t v[4] = {in[y].x, in[y].y, in[y].z, in[y].w};
    // largest magnitude of the group, as integers, as which they order alike; infinities and NaN come last
    uint32_t top = __vmaxu2(__vmaxu2(v[0] & 0x7fff7fffu, v[1] & 0x7fff7fffu), __vmaxu2(v[2] & 0x7fff7fffu, v[3] & 0x7fff7fffu));
    top = max(top & 0xffffu, top >> 16);
#pragma unroll
    for (int s = 1; s < GL; s <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, s));
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack2<T>(v[e]);
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
    // (a product with the nearest number to 1/7, 2^-26 of it away, rounds to bf16 as the quotient does: amax has 11 bits at most, so
    // amax / 7 is a number of 9 bits, which the product rounds to, or 2^-12 of itself from the middle of two bf16 numbers)
    const __nv_bfloat16 s16 = __float2bfloat16_rn(unpack2<T>(top).x * (1.f / 7.f));
    uint32_t sbits = *reinterpret_cast<const uint16_t*>(&s16);
    if (sbits < 0x0080u) sbits = 0u;  // below the smallest normal number
    // Codes c + 8 by one fma each, in the low bits of a sum with 2^23: with the quotients moved by 2^-20 of themselves there is
    // no half to be rounded, and the nearest number is the definition's.  (s 0: the quotients are 0.)
    float inv = sbits != 0u ? fast_rcp(__uint_as_float(sbits << 16)) * (1.f + 9.5367431640625e-7f) : 0.f;
    if (top >= kInfinity) {
      sbits = 0xffc0u;
      inv = 0.f;
    }
    uint32_t word = __float_as_uint(fmaf(x[7], inv, 8388616.f));
#pragma unroll
    for (int e = 6; e >= 0; --e) word = word * 16u + __float_as_uint(fmaf(x[e], inv, 8388616.f));
    word -= 0xfb000000u;  // what is left of 2^23, 0x4b000000 in elements 0 and 1
    if (D >= 32) word = VALUES ? exchange_halves<D>(rotate_halves(word), w, true) : __funnelshift_l(word, word, 2);
    if (WHOLE || place.real(m)) {
      const int64_t row = WHOLE ? row0 + y * lanes : place.at(m, bad);
      if (WHOLE || row >= 0) {
        *reinterpret_cast<uint32_t*>(codes + row * (D / 2)) = word;
        if (w % GL == 0) scales[row * NG] = (uint16_t)sbits;
      }
    }
  }
}

template <typename T, int D, bool VALUES, bool WHOLE, int EACH>
__device__ __forceinline__ void read_rows(const CacheParams& c, const CacheRows& r, const RowPlace& place, const RowTile& t, bool* bad) {
  constexpr int TPR = D / 8, NG = D >= 32 ? D / 32 : 1, GL = D >= 32 ? 4 : 2;
  const int w = threadIdx.x % TPR, lanes = t.lanes, m0 = t.first + threadIdx.x / TPR;
  // WHOLE: the rows lie one behind the other
  const int64_t row0 = WHOLE ? place.at(m0, bad) : 0;
  const unsigned char* codes =
      static_cast<const unsigned char*>(VALUES ? c.v_codes : c.k_codes) + (D >= 32 && !VALUES ? (w % 4) * NG + w / 4 : w) * 4;
  const uint16_t* scales = static_cast<const uint16_t*>(VALUES ? c.v_scales : c.k_scales) + w / GL;
  uint32_t words[EACH], sbits[EACH];
#pragma unroll
  for (int y = 0; y < EACH; ++y) {
    const int m = m0 + y * lanes;
    words[y] = D >= 32 ? 0x22222222u : 0x88888888u;  // padding: zeros
    sbits[y] = 0u;
    if (WHOLE || place.real(m)) {
      const int64_t row = WHOLE ? row0 + y * lanes : place.at(m, bad);
      sbits[y] = 0xffc0u;
      if (WHOLE || row >= 0) {
        words[y] = *reinterpret_cast<const uint32_t*>(codes + row * (D / 2));
        sbits[y] = scales[row * NG];
      }
    }
  }
  const int64_t ss = r.ss[VALUES];
  T* dst = static_cast<T*>(r.dst[VALUES]) + t.b * r.sb[VALUES] + t.hk * r.sh[VALUES] + m0 * ss + w * 8;
#pragma unroll
  for (int y = 0; y < EACH; ++y) {
    uint32_t word = words[y];
    if (D >= 32) word = VALUES ? rotate_halves_back(exchange_halves<D>(word, w, false)) : __funnelshift_r(word, word, 2);
    // elements (0, 4), (1, 5), (2, 6), (3, 7), each exact as a 16-bit number; their products are rounded once
    uint32_t pair[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) pair[e] = code_times_scale<T>(word >> (4 * e) & 0x000f000fu, sbits[y]);
    const uint4 out = make_uint4(__byte_perm(pair[0], pair[1], 0x5410), __byte_perm(pair[2], pair[3], 0x5410),
                                 __byte_perm(pair[0], pair[1], 0x7632), __byte_perm(pair[2], pair[3], 0x7632));
    if (WHOLE || m0 + y * lanes < r.rows) {
      T* to = dst + y * lanes * ss;
      if (WHOLE || r.vec) *reinterpret_cast<uint4*>(to) = out;
      else {
        const uint32_t o[4] = {out.x, out.y, out.z, out.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(o[e / 2] >> (16 * (e & 1)));
      }
    }
  }
  // Rows behind the table, zeros so far.  (Told apart where words are fetched they cost every call: 3 x 1531 rows of 12 heads of 64,
  // fp16, pages of 16: 6.8 us, 5.6 so.)
  if (!WHOLE && place.stop < r.rows) {
#pragma unroll 1
    for (int y = 0; y < EACH; ++y) {
      const int m = m0 + y * lanes;
      if (m < place.stop || m >= r.rows) continue;
#pragma unroll 1
      for (int e = 0; e < 8; ++e) reinterpret_cast<uint16_t*>(dst + y * lanes * ss)[e] = 0x7fffu;
    }
  }
}

// Keys in the first half of the grid, values in the second.  CTAs whose rows all exist, on one page, with 16-byte accesses, go
// without the checks for each row (4 sequences of 8192 rows of 8 heads of 128, inputs not in L2: bf16 and fp16 written in 38.9 us, read
// in 35.6 and 38.9; with the checks 45.1, 52.0 and 55.3).
template <typename T, int D, bool WRITE, int EACH>
__global__ void __launch_bounds__(256) cache_rows_kernel(const CacheParams c, const CacheBatch bt, const CacheRows r, int* status) {
  griddep_wait();
  griddep_launch_dependents();
  RowTile t;
  const int bh = blockIdx.x / (unsigned)r.tiles;
  t.b = bh / (unsigned)c.Hk;
  t.hk = bh - t.b * c.Hk;
  t.lanes = blockDim.x / (D / 8);
  const int rows = t.lanes * EACH;
  t.first = (blockIdx.x - bh * r.tiles) * rows;
  bool bad = false;
  const RowPlace place = row_place(c, bt, r.rows, t.b, t.hk, t.first, t.first + rows, &bad);
  const bool whole = r.vec && t.first + rows <= place.stop && place.first + t.first >= 0 && (unsigned)place.one < (unsigned)c.pages;
  auto run = [&](auto values, auto all) {
    if constexpr (WRITE) write_rows<T, D, decltype(values)::value, decltype(all)::value, EACH>(c, r, place, t, &bad);
    else read_rows<T, D, decltype(values)::value, decltype(all)::value, EACH>(c, r, place, t, &bad);
  };
  if (blockIdx.y == 0) {
    if (whole) run(std::false_type{}, std::true_type{});
    else run(std::false_type{}, std::false_type{});
  } else {
    if (whole) run(std::true_type{}, std::true_type{});
    else run(std::true_type{}, std::false_type{});
  }
  if (bad && status != nullptr) atomicOr(status, kBadPage);
}

// ---------------------------------------------------------------------------------------------- attention
// One kv head's rows (the M query rows of each of its G query heads, one head after the other), 8 at a time,
// against the tokens they see, in tiles of 128.  The bytes of the cache bound it, so the tiles of all sequences and heads
// are one list that is cut into equal shares, a CTA each: lengths are on the device, and no share waits for the longest
// sequence.  What a share has of an item (a row block) that it does not finish goes to the workspace, and a second kernel
// adds up the parts of each item in order.
//   warp 4      brings tiles into shared memory: codes and scales of a page and head are one bulk copy each
//   warps 0-3   take 32 tokens of a tile each, with a running maximum, sum and output of their own, merged at the end
// Matrix instructions are mma.sync m16n8k16 in fp16: a tile has 8 rows, and the operands come out of registers, where
// a nibble n in bits 2..5 of a half IS the number n 2^-22 (a subnormal): unpacking is one AND per pair, one rotation
// per two.  Nibbles in bits 6..9 are 16 n 2^-22: the query's elements there (the output's rows there) carry 1/16.  The
// matrix instructions align a subnormal as they do 2^-14, so that its products keep 2^-16 of a code, for nibbles in bits 6..9
// 2^-20; with nibbles in bits 0..3 and 4..7 it would be 2^-14 and 2^-18.
//   S = sum_g s_g (sum_d q_d n_d - 8 sum_d q_d)    per group g of the key: the scale multiplies the fp32 product, the sum of
//                                                  q comes in as the accumulator's start.  q is moved by a power of two per
//                                                  row to just below 2^15, so that fp16 holds bf16 queries too.
//   O_d = sum_j (P_j s_jg) (n_jd - 8)              the scale of the value goes onto the weight; -8 comes by another matrix instruction
//                                                  with the same rounded weights, 16 tokens at a time: summed apart, the two would
//                                                  grow with the tokens and lose in their difference what long contexts average out
//                                                  (64 x 16384 tokens, fp16: 3.3e-4 of the output against 2.9e-4).
// Weights are fp16: 2^-11 of each.  The running maximum is that of S + log2 s, s the largest scale of the token's value, so that
// P s stays within fp16 for values of any size.  Below 2^-14 of the largest P s weights are subnormal and off by up to 2^-25 of it:
// one maximum for all groups of 32 channels, so a group of values a power of two below its neighbours has as many bits less there.
constexpr int RT = 8;         // rows of a row block: the width of a matrix instruction
constexpr int TT = 128;       // tokens of a tile
constexpr int STAGES = 3;
constexpr int CONSUMERS = 4;  // warps
constexpr int CTA_THREADS = 32 * (CONSUMERS + 1);
constexpr int CTAS_PER_SM = 3;
constexpr uint32_t kLow = 0x003c003cu, kHigh = 0x03c003c0u;  // the two nibbles of each half's mantissa

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Without an accumulator to begin with.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// 8 x 8 halves across a warp: on entry lane 4 i + j has elements (i, 2 j) and (i, 2 j + 1), on exit (2 j, i) and (2 j + 1, i).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Barrier of the consumer warps; whether any thread said so.
__device__ __forceinline__ bool consumers_any(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)mine), "n"(32 * CONSUMERS)
      : "memory");
  return any != 0;
}

// Tokens of sequence b that the table has no room for.  (Read where it is wanted: kept, it would be spilled.)
__device__ __forceinline__ int tokens_beyond(const CacheAttnParams& p, int b) {
  return max(0, p.batch.lengths[b] - table_room(p.batch, p.cache.page_shift));
}
// Tiles that the rows of a sequence see: [0, ns), then [w0, w0 + nt - ns).  `len`: the tokens that the table has room for.
struct Span {
  int len, lo, ns, w0, nt;
  __device__ __forceinline__ int tile(int it) const { return it < ns ? it : w0 + it - ns; }
};
__device__ __forceinline__ Span span_of(const CacheAttnParams& p, int b, bool* bad) {
  Span s;
  const int room = table_room(p.batch, p.cache.page_shift);
  const int end = told_length(p.batch, room, b, bad);
  s.len = min(end, room);
  // the first key that the first row's window has (the last one where there is none: a sequence with keys has a tile)
  s.lo = max(0, min(end - p.M - p.window + 1, s.len - 1));
  s.w0 = s.lo / TT;
  s.ns = min((min(p.sinks, s.len) + TT - 1) / TT, s.w0);
  s.nt = s.len > 0 ? s.ns + (s.len + TT - 1) / TT - s.w0 : 0;
  return s;
}

// The tiles of all items (b, kv head, row block) in a row, cut into `shares` that differ by one at most.  (The entry point keeps
// the list below 2^31 tiles.)
struct Shares {
  int shares, per, more;  // the first `more` shares have one tile more
  Shares() = default;
  __device__ __forceinline__ Shares(const CacheAttnParams& p, int total) {
    shares = max(1, min(p.grid, total));
    per = total / shares;
    more = total - per * shares;
  }
  __device__ __forceinline__ int begin(int c) const { return c * per + min(c, more); }
  __device__ __forceinline__ int of(int tile) const {
    const int cut = more * (per + 1);
    return tile < cut ? tile / (per + 1) : more + (tile - cut) / per;
  }
};

// A share's walk over its segments, each some tiles of one item.
struct Walk {
  int at, end;  // in the list of tiles
  int b, item;  // item: kv head * row_blocks + row block
  int first;    // first tile of the segment within its item
  Span span;
  __device__ __forceinline__ int count() const { return min(span.nt - first, end - at); }
};
// The CTA's first segment, by one warp.  false: the share is empty.
__device__ __forceinline__ bool walk_begin(const CacheAttnParams& p, int lane, Walk* w, Shares* shares) {
  const int items = p.cache.Hk * p.row_blocks;
  bool bad = false;
  int total = 0, n = 0;  // n: tiles of the sequences of a chunk of 32 up to this lane's
  auto chunk = [&](int b0) {
    n = b0 + lane < p.batch.B ? span_of(p, b0 + lane, &bad).nt * items : 0;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, n, s);
      if (lane >= s) n += up;
    }
    return __shfl_sync(0xffffffffu, n, 31);
  };
  for (int b0 = 0; b0 < p.batch.B; b0 += 32) total += chunk(b0);
  if (bad && p.status != nullptr) atomicOr(p.status, kBadPage);
  const Shares sh(p, total);
  *shares = sh;
  w->at = sh.begin(min((int)blockIdx.x, sh.shares));
  w->end = sh.begin(min((int)blockIdx.x + 1, sh.shares));
  if (w->at >= w->end) return false;
  int base = 0;
  // (lengths that change under the call, which they must not, end the walk here or in walk_next, not the batch)
  for (int b0 = 0; b0 < p.batch.B; b0 += 32) {
    const int all = p.batch.B <= 32 ? total : chunk(b0);  // (one chunk: as it was)
    const unsigned past = __ballot_sync(0xffffffffu, base + n > w->at);
    if (past != 0u) {
      const int first = __ffs(past) - 1;
      const int before = __shfl_sync(0xffffffffu, n, max(first - 1, 0));
      w->b = b0 + first;
      w->span = span_of(p, w->b, &bad);
      const int off = w->at - base - (first == 0 ? 0 : before);
      w->item = off / max(w->span.nt, 1);
      w->first = off - w->item * w->span.nt;
      return w->span.nt > 0 && w->item < items;
    }
    base += all;
  }
  return false;
}
__device__ __forceinline__ bool walk_next(const CacheAttnParams& p, Walk* w, volatile int* abort_flag) {
  w->at += w->count();
  if (w->at >= w->end) return false;
  w->first = 0;
  if (++w->item >= p.cache.Hk * p.row_blocks) {
    w->item = 0;
    bool bad = false;
    do {
      if (++w->b >= p.batch.B) {  // (the list has more tiles, so a later sequence has some)
        *abort_flag = 1;
        return false;
      }
      w->span = span_of(p, w->b, &bad);
    } while (w->span.nt == 0);
  }
  return true;
}

template <int D>
struct CacheSmem {
  static constexpr int NG = D >= 32 ? D / 32 : 1;
  static constexpr int kRow = D / 2, kScale = NG * 2;  // bytes of a token
  static constexpr int k_off = 0, v_off = TT * kRow, ks_off = 2 * TT * kRow, vs_off = ks_off + TT * kScale;
  static constexpr int kStage = vs_off + TT * kScale;
  static constexpr int out_off = STAGES * kStage;  // CONSUMERS x RT x (D + 4) floats, then (m, l) of them
  static constexpr int kOutRow = D + 4;
  static constexpr int ml_off = out_off + CONSUMERS * RT * kOutRow * 4;
  static constexpr int bar_off = ml_off + CONSUMERS * RT * 8;
  // While a segment lasts a warp's part of the output area holds its 32 tokens' scales of keys and values as pairs of floats.
  static_assert(2 * 32 * NG * 8 <= RT * kOutRow * 4, "room for the scales");
  static constexpr int total = bar_off + 192;
};
struct CacheBars {
  uint64_t full[STAGES], empty[STAGES];
  int abort_flag, any;
  Walk walk;  // where the CTA begins
  Shares shares;
};
static_assert(sizeof(CacheBars) <= 192, "room for the barriers");

// Workspace: a header per share, then two slots of RT rows: D floats, the row's maximum (log2 units) and sum, and 2 floats unused.
// Slot 0: the share's first segment, where it does not begin its item; slot 1: the last, where it begins its item but does not
// end it.  The header tells what slot 1 is the beginning of: sequence, item, and the share that ends it, -1 where there is none.
template <int D>
__device__ __forceinline__ float* part_slot(const CacheAttnParams& p, int share, int slot) {
  return p.parts + p.grid * 4 + ((int64_t)share * 2 + slot) * RT * (D + 4);
}
__device__ __forceinline__ int4* part_header(const CacheAttnParams& p, int share) { return reinterpret_cast<int4*>(p.parts) + share; }

// Four elements of a finished row: sum / den, zeros for a row that saw nothing, NaN for the last `beyond` rows of a head, whose
// own keys lie behind the table.
template <typename T>
__device__ __forceinline__ void store_row(const CacheAttnParams& p, int b, int beyond, int hk, int r, int d, float4 sum, float top,
                                          float den) {
  if (r >= p.rows) return;
  const int head = hk * p.G + r / p.M, i = r % p.M;
  if (i >= p.M - beyond) den = __int_as_float(0x7fffffff);
  const float inv = den == 0.f ? 0.f : 1.f / den;  // (a NaN stays one)
  T* dst = static_cast<T*>(p.out) + b * p.o_sb + (int64_t)head * p.o_sh + (int64_t)i * p.o_ss + d;
  const uint32_t lo = pack2<T>(sum.x * inv, sum.y * inv), hi = pack2<T>(sum.z * inv, sum.w * inv);
  if (p.vec_out) *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
  else {
    uint16_t* e = reinterpret_cast<uint16_t*>(dst);
    e[0] = (uint16_t)lo; e[1] = (uint16_t)(lo >> 16); e[2] = (uint16_t)hi; e[3] = (uint16_t)(hi >> 16);
  }
  if (d == 0 && p.L != nullptr)
    p.L[((int64_t)b * p.G * p.cache.Hk + head) * p.M + i] = den == 0.f ? FAWS_NEG_INF : fmaf(top, kLn2, logf(den));
}

template <typename T, int D>
__global__ void __launch_bounds__(CTA_THREADS, CTAS_PER_SM) cache_attn_kernel(const CacheAttnParams p) {
  using L = CacheSmem<D>;
  constexpr int NG = L::NG;
  constexpr int MT = D >= 32 ? 2 : 1;  // 16-row tiles of a group's output
  extern __shared__ __align__(128) unsigned char smem[];
  CacheBars* bars = reinterpret_cast<CacheBars*>(smem + L::bar_off);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&bars->full[s], 32);
      mbar_init(&bars->empty[s], CONSUMERS);
    }
    bars->abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  // nothing to join, until this thread says so (a share whose waits give up may not come to that)
  if (threadIdx.x == 0) part_header(p, blockIdx.x)->w = -1;
  if (warp == 0) {
    Walk first;
    Shares shares;
    const bool some = walk_begin(p, lane, &first, &shares);
    if (lane == 0) {
      bars->any = some ? 1 : 0;
      bars->walk = first;
      bars->shares = shares;
    }
  } else if (warp == 1) {
    // Sequences without a key have no tiles: their rows are zero.  A sequence's rows are shared by as many CTAs as leave each 64
    // stores of a warp, one where a sequence has few rows (two sequences of 2048 rows, 32 heads of 128, one of them empty: 11.7 ms
    // with one CTA for it).
    constexpr int kLanes = D / 4, kRows = 32 / kLanes;  // lanes of a row, rows of a warp
    const int parts = (int)min((int64_t)gridDim.x, ((int64_t)p.cache.Hk * p.rows + 64 * kRows - 1) / (64 * kRows));
    for (int64_t y = blockIdx.x; y < (int64_t)p.batch.B * parts; y += gridDim.x) {
      const int b = (int)(y / parts), part = (int)(y - (int64_t)b * parts);
      bool bad = false;
      if (span_of(p, b, &bad).nt > 0) continue;
      for (int hk = 0, r = part * kRows + lane / kLanes;; r += parts * kRows) {
        for (; r >= p.rows && hk < p.cache.Hk; ++hk) r -= p.rows;
        if (hk >= p.cache.Hk) break;
        store_row<T>(p, b, 0, hk, r, lane % kLanes * 4, make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f);
      }
    }
  }
  __syncthreads();
  const bool any = bars->any != 0;
  Walk w = bars->walk;

  if (any && warp == CONSUMERS) {
    // ------------------------------------------------------------ copies
    // A lane's copy: one of the four arrays (codes and scales of keys and values) of one of up to 8 pieces of the tile, a piece
    // being what a page has of it.  Only tokens that some row may see are copied, 16 at a time (both ends of a copy lie on 16
    // bytes then); what a stage holds elsewhere is never used.
    const int kind = lane & 3;
    const int shift = min(p.cache.page_shift, 7), piece = lane >> 2;  // tokens of a piece: 1 << shift
    const bool mine = piece < TT >> shift;
    const int bytes = kind < 2 ? L::kRow : L::kScale;
    const int off = kind == 0 ? L::k_off : kind == 1 ? L::v_off : kind == 2 ? L::ks_off : L::vs_off;
    const unsigned char* src = static_cast<const unsigned char*>(kind == 0   ? p.cache.k_codes
                                                                 : kind == 1 ? p.cache.v_codes
                                                                 : kind == 2 ? p.cache.k_scales
                                                                             : p.cache.v_scales);
    // what of tile `it` of the segment this lane copies, and the page that has it
    struct Piece {
      int t0, lo, hi, page;
    };
    auto piece_of = [&](int it) -> Piece {
      Piece c;
      c.t0 = w.span.tile(w.first + it) * TT;
      // what may be seen of the tile: the sinks, the windows, or both
      c.lo = max(c.t0, w.span.lo);
      c.hi = min(c.t0 + TT, w.span.len);
      if (c.t0 < p.sinks) {
        if (c.lo >= c.hi) c.hi = min(c.hi, p.sinks);
        c.lo = c.t0;
      }
      const int p0 = c.t0 + (piece << shift);
      c.lo = max(c.lo, p0) & ~15;
      c.hi = min((min(c.hi, p0 + (1 << shift)) + 15) & ~15, p0 + (1 << shift));
      c.page = -1;
      if (!mine) c.hi = c.lo;
      if (c.lo < c.hi) c.page = p.batch.table[(int64_t)w.b * p.batch.table_stride + (p0 >> p.cache.page_shift)];
      return c;
    };
    int n = 0;  // tiles so far
    bool ok = true, bad = false;
    do {
      const int hk = w.item / p.row_blocks, cnt = w.count();
      Piece next = piece_of(0);
      for (int it = 0; ok && it < cnt; ++it, ++n) {
        const Piece c = next;
        if (it + 1 < cnt) next = piece_of(it + 1);  // (its page comes while the tile before it waits for room)
        const int s = n % STAGES;
        if (lane == 0) ok = n < p.tiles_at_most && mbar_wait(&bars->empty[s], ((n / STAGES) & 1) ^ 1, abort_flag, p.wait_cycles);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        unsigned char* dst = smem + s * L::kStage + off + (c.lo - c.t0) * bytes;
        const int size = (c.hi - c.lo) * bytes;
        if (size > 0 && (unsigned)c.page < (unsigned)p.cache.pages) {
          mbar_arrive_expect_tx(&bars->full[s], size);
          const int64_t row = (((int64_t)c.page * p.cache.Hk + hk) << p.cache.page_shift) + (c.lo & ((1 << p.cache.page_shift) - 1));
          bulk_load_1d(dst, src + row * bytes, size, &bars->full[s]);
        } else {
          if (size > 0) {  // a page that does not exist: its keys are NaN
            bad = true;
            if (kind == 2) {
              for (int x = 0; x < size; x += 4) *reinterpret_cast<uint32_t*>(dst + x) = 0xffc0ffc0u;
              fence_proxy_async_smem();  // (later copies go over them)
            }
          }
          mbar_arrive(&bars->full[s]);
        }
      }
    } while (ok && walk_next(p, &w, abort_flag));
    if (bad && p.status != nullptr) atomicOr(p.status, kBadPage);
  } else if (any) {
    // ------------------------------------------------------------ rows
    // Scores are taken with keys as rows of the matrix instructions and queries as columns, outputs with elements as rows and
    // queries as columns: 8 rows are an instruction's whole width.  Row i of 16 keys is token token_of(i) of the 16, an order in
    // which the loads of keys meet no bank twice.  A lane's scores are those of tokens g and g + 8 with rows 2 t and 2 t + 1 (of 8);
    // weights turn from there into columns' operands by movmatrix.
    const int g = lane >> 2, t = lane & 3;
    const int krow = (g & 1) ? ((g >> 1) ^ 1) + 4 : g >> 1;      // token_of(g); token_of(i + 8) = token_of(i) + 8
    const int tok[4] = {t, (t ^ 1) + 4, t + 8, (t ^ 1) + 12};    // token_of(2 t), (2 t + 1), (2 t + 8), (2 t + 9)
    // -8 in every place, kept in registers: as a constant it is put there again for each product
    uint32_t less8[4];
    asm volatile("mov.b32 %0, 0x80208020;\n\tmov.b32 %1, 0x82008200;\n\tmov.b32 %2, 0x80208020;\n\tmov.b32 %3, 0x82008200;"
                 : "=r"(less8[0]), "=r"(less8[1]), "=r"(less8[2]), "=r"(less8[3]));
    float* so = reinterpret_cast<float*>(smem + L::out_off) + warp * RT * L::kOutRow;
    float4* table = reinterpret_cast<float4*>(so);  // [keys, values][pair of groups][token]
    float2* ml = reinterpret_cast<float2*>(smem + L::ml_off);
    int n = 0;
    bool ok = true;
    do {
      const int hk = w.item / p.row_blocks, r0 = (w.item % p.row_blocks) * RT, cnt = w.count();
      const int end = w.span.len + tokens_beyond(p, w.b);  // one behind the last row's position
      // ---- the rows' queries as fp16 operands, and -8 sum of each group; a lane loads row g of 8
      uint32_t q[NG][2][2];
      uint64_t qbias[NG];    // of rows 2 t and 2 t + 1, as f
      float f[2];
      int hi_row[2];         // a row sees keys [hi_row - window, hi_row) and the sinks before hi_row
      {
        const int r = r0 + g;
        const bool real = r < p.rows;
        const int head = r / p.M, i = r - head * p.M;
        float x[NG][8];
        float top = 0.f;
        const T* qp = static_cast<const T*>(p.q) + w.b * p.q_sb + (int64_t)(hk * p.G + head) * p.q_sh + (int64_t)i * p.q_ss;
#pragma unroll
        for (int gi = 0; gi < NG; ++gi)
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const int d = D >= 32 ? 32 * gi + 8 * t + y : 4 * t + y;
            x[gi][y] = real && (D >= 32 || y < 4) ? to_f(qp[d]) : 0.f;
            top = fmaxf(top, fabsf(x[gi][y]));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int k = 14 - ((int)(__float_as_uint(top) >> 23) - 127);  // top goes to [2^14, 2^15)
        if (!(top > 0.f) || top >= __int_as_float(0x7f800000)) k = 0;
        k = max(-100, min(100, k));
        const float mul = __int_as_float((127 + k) << 23);
        // 2^22 undoes the subnormal; in two factors, so that neither leaves fp32's range
        const float my_f = p.sm_scale * kLog2e * __int_as_float((127 + 22) << 23) * __int_as_float((127 - k) << 23);
        const int my_hi = real ? end - p.M + i + 1 : 0;
        // rows 2 t and 2 t + 1 are loaded by the lanes 8 t and 8 t + 4
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          f[c] = __shfl_sync(0xffffffffu, my_f, 8 * t + 4 * c);
          hi_row[c] = __shfl_sync(0xffffffffu, my_hi, 8 * t + 4 * c);
        }
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          float sum = 0.f;
          __half h[8];
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            h[y] = __float2half_rn(x[gi][y] * mul * ((y & 1) ? 0.0625f : 1.f));
            sum += __half2float(h[y]) * ((y & 1) ? 16.f : 1.f);
          }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          sum *= -8.f * 2.384185791015625e-7f;
          qbias[gi] = pack_f32x2(__shfl_sync(0xffffffffu, sum, 8 * t), __shfl_sync(0xffffffffu, sum, 8 * t + 4));
          auto pair = [&](int a, int b) {
            return (uint32_t)__half_as_ushort(h[a]) | (uint32_t)__half_as_ushort(h[b]) << 16;
          };
          // element y of a word is nibble y: registers (0, 4), (1, 5), (2, 6), (3, 7)
          q[gi][0][0] = pair(0, 4);
          q[gi][0][1] = pair(1, 5);
          q[gi][1][0] = pair(2, 6);
          q[gi][1][1] = pair(3, 7);
        }
      }
      float o[NG][MT][4], m[2], l[2];
      m[0] = m[1] = FAWS_NEG_INF;
      l[0] = l[1] = 0.f;
#pragma unroll
      for (int gi = 0; gi < NG; ++gi)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) o[gi][mt][c] = 0.f;
      // of the first, the last row (rows whose own key is behind `len` become NaN, whatever they take part in)
      const int hi_first = end - p.M + 1, lo_last = end - p.window;

      // ---- 32 tokens from `base` of the stage on, the first of them at position n0, in two parts of 16; their scores come first, so
      // that the maximum is looked at once
      auto step = [&](auto masked_tag, const unsigned char* stage, int base, int n0) {
        constexpr bool kMasked = decltype(masked_tag)::value;
        // Each lane converts one token's scales, each number twice, as the packed products want them.  Of the value scales also
        // log2 of the token's largest, no less than -100 (a NaN, negative as an integer, has none).
        float my_ev;
        {
          int top = 0x0d800000;  // 2^-100
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const unsigned char* sp = stage + (kv ? L::vs_off : L::ks_off) + (base + lane) * L::kScale;
            using Entry = typename std::conditional<NG == 1, float2, float4>::type;
            Entry* to = reinterpret_cast<Entry*>(table) + kv * 32 * ((NG + 1) / 2) + lane;
            auto twice = [](uint32_t w) { return make_float4(bf16_lo(w), bf16_lo(w), bf16_hi(w), bf16_hi(w)); };
            if constexpr (NG == 4) {
              const uint2 w2 = *reinterpret_cast<const uint2*>(sp);
              to[0] = twice(w2.x);
              to[32] = twice(w2.y);
              if (kv) {
                const uint32_t mx = __vmaxs2(w2.x, w2.y);
                top = max(max((int)(mx << 16), (int)(mx & 0xffff0000u)), top);
              }
            } else if constexpr (NG == 2) {
              const uint32_t w1 = *reinterpret_cast<const uint32_t*>(sp);
              to[0] = twice(w1);
              if (kv) top = max(max((int)(w1 << 16), (int)(w1 & 0xffff0000u)), top);
            } else {
              const uint32_t w1 = (uint32_t)*reinterpret_cast<const uint16_t*>(sp) << 16;
              to[0] = make_float2(__uint_as_float(w1), __uint_as_float(w1));
              if (kv) top = max((int)w1, top);
            }
          }
          my_ev = fast_log2(__int_as_float(top));
        }
        __syncwarp();
        // scales (s, s) of the token `at` of the 32, group by group
        auto scales = [&](int kv, int at, uint64_t (&sc)[NG]) {
          if constexpr (NG >= 2) {
            const float4* from = table + kv * 32 * (NG / 2) + at;
#pragma unroll
            for (int gi = 0; gi < NG; gi += 2) {
              const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(from + gi / 2 * 32);
              sc[gi] = x.x;
              sc[gi + 1] = x.y;
            }
          } else sc[0] = reinterpret_cast<const uint64_t*>(table)[kv * 32 + at];
        };
        // scores without the rows' factors f: [part][rows 2 t, 2 t + 1][token g, g + 8]
        uint64_t s[2][2];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t kw[2][NG];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const unsigned char* kr = stage + L::k_off + (base + part * 16 + half * 8 + krow) * L::kRow;
            if constexpr (NG == 4) *reinterpret_cast<uint4*>(kw[half]) = *reinterpret_cast<const uint4*>(kr + t * 16);
            else if constexpr (NG == 2) *reinterpret_cast<uint2*>(kw[half]) = *reinterpret_cast<const uint2*>(kr + t * 8);
            else if constexpr (D == 32) kw[half][0] = *reinterpret_cast<const uint32_t*>(kr + t * 4);
            else kw[half][0] = (uint32_t)*reinterpret_cast<const uint16_t*>(kr + t * 2) << 2;  // elements 4 t .. + 3, then none
          }
          uint64_t sc[2][NG];
          scales(0, part * 16 + krow, sc[0]);
          scales(0, part * 16 + 8 + krow, sc[1]);
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            const uint32_t y0 = __funnelshift_r(kw[0][gi], kw[0][gi], 8), y1 = __funnelshift_r(kw[1][gi], kw[1][gi], 8);
            const uint32_t a0[4] = {kw[0][gi] & kLow, kw[1][gi] & kLow, kw[0][gi] & kHigh, kw[1][gi] & kHigh};
            const uint32_t a1[4] = {y0 & kLow, y1 & kLow, y0 & kHigh, y1 & kHigh};
            float acc[4];
            mma_f16_first(acc, a0, q[gi][0][0], q[gi][0][1]);
            mma_f16(acc, a1, q[gi][1][0], q[gi][1][1]);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint64_t x = add_f32x2(pack_f32x2(acc[2 * half], acc[2 * half + 1]), qbias[gi]);
              s[part][half] = gi == 0 ? mul_f32x2(x, sc[half][gi]) : fma_f32x2(x, sc[half][gi], s[part][half]);
            }
          }
        }
        // ---- running maximum, moved only when a weighted value would exceed 2^8
        [[maybe_unused]] uint32_t hidden;  // bit 4 part + 2 half + row
        float top[2], ev[2][2];
        bool need = false;
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int half = 0; half < 2; ++half) ev[part][half] = __shfl_sync(0xffffffffu, my_ev, part * 16 + half * 8 + krow);
        hidden = 0u;
        float x[2][2][2];
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float y[2];
            unpack_f32x2(s[part][half], y[0], y[1]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              x[c][part][half] = fmaf(y[c], f[c], ev[part][half]);
              if constexpr (kMasked) {
                const int j = n0 + part * 16 + half * 8 + krow;
                if (!(j < hi_row[c] && (j >= hi_row[c] - p.window || j < p.sinks))) {
                  x[c][part][half] = FAWS_NEG_INF;
                  hidden |= 1u << (part * 4 + half * 2 + c);
                }
              }
            }
          }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[c] = fmax3(fmaxf(x[c][0][0], x[c][0][1]), x[c][1][0], x[c][1][1]);
          need = need || top[c] > m[c] + 8.f;
        }
        if (__any_sync(0xffffffffu, need)) {
          float alpha[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = top[c];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            const float m_new = fmaxf(m[c], mx);
            alpha[c] = m_new == FAWS_NEG_INF ? 1.f : fast_exp2(m[c] - m_new);
            m[c] = m_new;
            l[c] *= alpha[c];
          }
#pragma unroll
          for (int gi = 0; gi < NG; ++gi)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) o[gi][mt][c] *= alpha[c & 1];
        }
        // ---- weights, and values
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint64_t pr[2];  // [token g, g + 8], rows 2 t and 2 t + 1
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float y[2];
            unpack_f32x2(s[part][half], y[0], y[1]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              y[c] = fast_exp2(fmaf(y[c], f[c], m[c] == FAWS_NEG_INF ? 0.f : -m[c]));
              if (kMasked && (hidden >> (part * 4 + half * 2 + c) & 1u)) y[c] = 0.f;
              l[c] += y[c];
            }
            pr[half] = pack_f32x2(y[0], y[1]);
          }
          uint64_t vs[2][NG];
          scales(1, part * 16 + krow, vs[0]);
          scales(1, part * 16 + 8 + krow, vs[1]);
          uint32_t vw[4][(NG + 1) / 2];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned char* vr = stage + L::v_off + (base + part * 16 + tok[e]) * L::kRow;
            if constexpr (NG == 4) *reinterpret_cast<uint2*>(vw[e]) = *reinterpret_cast<const uint2*>(vr + g * 8);
            else if constexpr (NG == 2) vw[e][0] = *reinterpret_cast<const uint32_t*>(vr + g * 4);
            else if constexpr (D == 32) vw[e][0] = *reinterpret_cast<const uint16_t*>(vr + g * 2);
            else vw[e][0] = vr[g];
          }
          // the weighted scales as operands, all of them before the products that wait for them
          uint32_t pb[NG][2];
#pragma unroll
          for (int gi = 0; gi < NG; ++gi)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float pv[2];
              unpack_f32x2(mul_f32x2(pr[half], vs[half][gi]), pv[0], pv[1]);
              if constexpr (kMasked) {  // a hidden token's scale may be anything
#pragma unroll
                for (int c = 0; c < 2; ++c)
                  if (hidden >> (part * 4 + half * 2 + c) & 1u) pv[c] = 0.f;
              }
              pb[gi][half] = transpose8(pack2<__half>(pv[0], pv[1]));
            }
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            // both tokens' half-words of the group; then with their bytes exchanged, which brings the next two nibbles
            const uint32_t sel = (gi & 1) ? 0x7632u : 0x5410u;
            [[maybe_unused]] const uint32_t swapped = (gi & 1) ? 0x6723u : 0x4501u;
            uint32_t x01 = __byte_perm(vw[0][gi >> 1], vw[1][gi >> 1], sel), x23 = __byte_perm(vw[2][gi >> 1], vw[3][gi >> 1], sel);
            if (D == 16) {
              x01 <<= 2;
              x23 <<= 2;
            }
            const uint32_t a0[4] = {x01 & kLow, x01 & kHigh, x23 & kLow, x23 & kHigh};
            [[maybe_unused]] uint32_t a1[4];
            if constexpr (MT == 2) {
              const uint32_t y01 = __byte_perm(vw[0][gi >> 1], vw[1][gi >> 1], swapped);
              const uint32_t y23 = __byte_perm(vw[2][gi >> 1], vw[3][gi >> 1], swapped);
              a1[0] = y01 & kLow; a1[1] = y01 & kHigh; a1[2] = y23 & kLow; a1[3] = y23 & kHigh;
            }
            mma_f16(o[gi][0], a0, pb[gi][0], pb[gi][1]);
            if constexpr (MT == 2) mma_f16(o[gi][MT - 1], a1, pb[gi][0], pb[gi][1]);
            mma_f16(o[gi][0], less8, pb[gi][0], pb[gi][1]);
            if constexpr (MT == 2) mma_f16(o[gi][MT - 1], less8, pb[gi][0], pb[gi][1]);
          }
        }
      };

      for (int it = 0; ok && it < cnt; ++it, ++n) {
        const int t0 = w.span.tile(w.first + it) * TT, st = n % STAGES;
        // (of one mind: the lanes of a warp go on together, or none)
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->full[st], (n / STAGES) & 1, abort_flag, p.wait_cycles));
        if (!ok) break;
        const unsigned char* stage = smem + st * L::kStage;
        const int n0 = t0 + warp * 32;
        const bool whole = n0 + 32 <= hi_first && (n0 >= lo_last || n0 + 32 <= p.sinks);
        // (32 tokens that no row sees are skipped)
        if (whole) step(std::false_type{}, stage, warp * 32, n0);
        else if (n0 < w.span.len && (n0 + 32 > w.span.lo || n0 < p.sinks)) step(std::true_type{}, stage, warp * 32, n0);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->empty[st]);
      }

      // ---- the four warps' parts
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float ls = l[c];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, x);
        if (g == 0) ml[warp * RT + 2 * t + c] = make_float2(m[c], ls);
      }
#pragma unroll
      for (int gi = 0; gi < NG; ++gi)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int row = 2 * t + (c & 1);
            const int d = D >= 32 ? 32 * gi + 4 * g + 2 * mt + (c >> 1) : 2 * g + (c >> 1);
            so[row * L::kOutRow + d] = o[gi][mt][c] * (c >> 1 ? 262144.f : 4194304.f);
          }
      consumers_any(false);
      const bool begins = w.first == 0, ends = w.first + cnt == w.span.nt;
      const float* all = reinterpret_cast<const float*>(smem + L::out_off);
      for (int x = threadIdx.x; x < RT * (D / 4); x += 32 * CONSUMERS) {
        const int row = x / (D / 4), d = (x % (D / 4)) * 4;
        float top = FAWS_NEG_INF;
#pragma unroll
        for (int c = 0; c < CONSUMERS; ++c) top = fmaxf(top, ml[c * RT + row].x);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
#pragma unroll
        for (int c = 0; c < CONSUMERS; ++c) {
          const float2 mlc = ml[c * RT + row];
          const float e = mlc.x == FAWS_NEG_INF ? 0.f : fast_exp2(mlc.x - top);
          const float4 v = *reinterpret_cast<const float4*>(all + (c * RT + row) * L::kOutRow + d);
          den = fmaf(e, mlc.y, den);
          sum.x = fmaf(e, v.x, sum.x); sum.y = fmaf(e, v.y, sum.y); sum.z = fmaf(e, v.z, sum.z); sum.w = fmaf(e, v.w, sum.w);
        }
        if (begins && ends) {
          store_row<T>(p, w.b, tokens_beyond(p, w.b), hk, r0 + row, d, sum, top, den);
        } else {
          float* part = part_slot<D>(p, blockIdx.x, begins ? 1 : 0) + row * (D + 4);
          *reinterpret_cast<float4*>(part + d) = sum;
          if (d == 0) *reinterpret_cast<float2*>(part + D) = make_float2(top, den);
        }
      }
      if (threadIdx.x == 0 && w.at + cnt >= w.end) {  // the share's last segment
        const int end = begins && !ends ? bars->shares.of(w.at + w.span.nt - 1) : -1;
        *part_header(p, blockIdx.x) = make_int4(w.b, w.item, 0, end);
      }
      ok = ok && walk_next(p, &w, abort_flag);
    } while (!consumers_any(!ok));  // (all of them go on, or none)
  }
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, 1);
    for (int x = 0; x < 50; ++x) __nanosleep(20000);  // let copies in flight land before the smem goes away
    __syncthreads();
  }
}

// The parts of the items that several shares had, added up in the order of the shares: a CTA per share, for the item that begins
// at its end.
template <typename T, int D>
__global__ void __launch_bounds__(256) cache_combine_kernel(const CacheAttnParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int c0 = blockIdx.x;
  const int4 head = *part_header(p, c0);
  const int c1 = head.w;
  if (c1 <= c0) return;
  // (no header of a call that ran to its end says anything else)
  if (c1 >= (int)gridDim.x || (unsigned)head.x >= (unsigned)p.batch.B || (unsigned)head.y >= (unsigned)(p.cache.Hk * p.row_blocks)) return;
  const int hk = head.y / p.row_blocks, r0 = (head.y % p.row_blocks) * RT;
  for (int x = threadIdx.x; x < RT * (D / 4); x += 256) {
    const int row = x / (D / 4), d = (x % (D / 4)) * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = FAWS_NEG_INF, den = 0.f;
    for (int c = c0; c <= c1; c += 4) {
      float4 v[4];
      float2 ml[4];
      float most = top;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        ml[y] = make_float2(FAWS_NEG_INF, 0.f);
        v[y] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c + y <= c1) {
          const float* part = part_slot<D>(p, c + y, c + y == c0 ? 1 : 0) + row * (D + 4);
          v[y] = *reinterpret_cast<const float4*>(part + d);
          ml[y] = *reinterpret_cast<const float2*>(part + D);
        }
        most = fmaxf(most, ml[y].x);
      }
      const float keep = top == FAWS_NEG_INF ? 0.f : fast_exp2(top - most);
      den *= keep;
      sum.x *= keep; sum.y *= keep; sum.z *= keep; sum.w *= keep;
      top = most;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float e = ml[y].x == FAWS_NEG_INF ? 0.f : fast_exp2(ml[y].x - most);
        den = fmaf(e, ml[y].y, den);
        sum.x = fmaf(e, v[y].x, sum.x); sum.y = fmaf(e, v[y].y, sum.y);
        sum.z = fmaf(e, v[y].z, sum.z); sum.w = fmaf(e, v[y].w, sum.w);
      }
    }
    store_row<T>(p, head.x, tokens_beyond(p, head.x), hk, r0 + row, d, sum, top, den);
  }
}

// A launch that may begin while the kernel before it drains (programmatic stream serialization).
template <typename K, typename... A>
cudaError_t launch_overlapped(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  count_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int D>
cudaError_t launch_attn_d(CacheAttnParams p, cudaStream_t s) {
  static PerDeviceOnce once;
  if (cudaError_t e = set_max_smem_once(once, cache_attn_kernel<T, D>, CacheSmem<D>::total); e != cudaSuccess) return e;
  p.row_blocks = (p.rows + RT - 1) / RT;
  if (p.tiles_at_most >= 0)
    if (cudaError_t e = launch_overlapped(cache_attn_kernel<T, D>, dim3(p.grid), CTA_THREADS, CacheSmem<D>::total, s, p); e != cudaSuccess)
      return e;
  return launch_overlapped(cache_combine_kernel<T, D>, dim3(p.grid), 256, 0, s, p);
}
template <typename T>
cudaError_t launch_attn_t(const CacheAttnParams& p, cudaStream_t s) {
  switch (p.cache.D) {
    case 16: return launch_attn_d<T, 16>(p, s);
    case 32: return launch_attn_d<T, 32>(p, s);
    case 64: return launch_attn_d<T, 64>(p, s);
    default: return launch_attn_d<T, 128>(p, s);
  }
}

int shares_at_most() { return CTAS_PER_SM * sm_count(); }

template <typename T, bool WRITE, int D>
cudaError_t launch_rows_d(const CacheParams& c, const CacheBatch& b, CacheRows r, cudaStream_t s) {
  // few rows (decoding): small CTAs, so that heads and sequences fill the chip
  const int each = r.rows * (D / 8) <= 256 ? 1 : kRowsEach;
  int lanes = 32 / (D / 8) > 1 ? 32 / (D / 8) : 1;
  while (lanes * (D / 8) < 256 && lanes * each < r.rows) lanes *= 2;
  r.tiles = (r.rows + lanes * each - 1) / (lanes * each);
  const dim3 grid((unsigned)((int64_t)b.B * c.Hk * r.tiles), 2, 1);
  return launch_overlapped(each == 1 ? cache_rows_kernel<T, D, WRITE, 1> : cache_rows_kernel<T, D, WRITE, kRowsEach>, grid,
                           lanes * (D / 8), 0, s, c, b, r, tc_status_word());
}
template <typename T, bool WRITE>
cudaError_t launch_rows_t(const CacheParams& c, const CacheBatch& b, const CacheRows& r, cudaStream_t s) {
  switch (c.D) {
    case 16: return launch_rows_d<T, WRITE, 16>(c, b, r, s);
    case 32: return launch_rows_d<T, WRITE, 32>(c, b, r, s);
    case 64: return launch_rows_d<T, WRITE, 64>(c, b, r, s);
    default: return launch_rows_d<T, WRITE, 128>(c, b, r, s);
  }
}

CacheRows make_rows(const faws_tensor* k, const faws_tensor* v, int rows, bool write) {
  CacheRows r{};
  const faws_tensor* t[2] = {k, v};
  r.vec = 1;
  for (int x = 0; x < 2; ++x) {
    if (write) r.src[x] = t[x]->ptr;
    else r.dst[x] = t[x]->ptr;
    r.sb[x] = t[x]->stride_b;
    r.sh[x] = t[x]->stride_h;
    r.ss[x] = t[x]->stride_s;
    if (!ok16(t[x]->ptr, r.sb[x], r.sh[x], r.ss[x])) r.vec = 0;
  }
  r.rows = rows;
  return r;
}

}  // namespace

cudaError_t launch_cache_write(const CacheParams& c, const CacheBatch& b, const faws_tensor* k, const faws_tensor* v, int rows,
                               int dtype, cudaStream_t s) {
  const CacheRows r = make_rows(k, v, rows, true);
  return dtype == FAWS_FP16 ? launch_rows_t<__half, true>(c, b, r, s) : launch_rows_t<__nv_bfloat16, true>(c, b, r, s);
}

cudaError_t launch_cache_read(const CacheParams& c, const CacheBatch& b, const faws_tensor* k, const faws_tensor* v, int rows,
                              int dtype, cudaStream_t s) {
  const CacheRows r = make_rows(k, v, rows, false);
  return dtype == FAWS_FP16 ? launch_rows_t<__half, false>(c, b, r, s) : launch_rows_t<__nv_bfloat16, false>(c, b, r, s);
}

size_t cache_attn_workspace_bytes(int D) { return (size_t)shares_at_most() * (16 + 2 * RT * (D + 4) * 4); }

cudaError_t launch_cache_attn(const CacheAttnParams& call, int dtype, cudaStream_t s) {
  CacheAttnParams p = call;
  p.grid = shares_at_most();
  p.vec_out = reinterpret_cast<uintptr_t>(p.out) % 8 == 0 && p.o_sb % 4 == 0 && p.o_sh % 4 == 0 && p.o_ss % 4 == 0;
  p.status = tc_status_word();
  return dtype == FAWS_FP16 ? launch_attn_t<__half>(p, s) : launch_attn_t<__nv_bfloat16>(p, s);
}

}  // namespace faws
