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

#include <algorithm>
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
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Length of sequence b as the cache can hold it; *bad where lengths says otherwise.
__device__ __forceinline__ int cached_length(const CacheBatch& c, int page_shift, int b, bool* bad) {
  const int n = c.lengths[b];
  const long long cap = (long long)c.max_pages << page_shift;
  const int most = cap > 0x3fffffff ? 0x3fffffff : (int)cap;
  if (n < 0 || n > most) *bad = true;
  return max(0, min(n, most));
}

// ---------------------------------------------------------------------------------------------- write, read
// A thread has 8 neighbouring elements of a row; D / 8 threads a row, the four (D 16: two) of a group next to each other.
// Bound by HBM: 2 bytes read and 9/16 written an element (read: the other way round).
struct CacheRows {
  const void* src[2];  // write: k, v; read: unused
  void* dst[2];        // read: k, v
  int64_t sb[2], sh[2], ss[2];
  int rows;            // of each sequence
  int vec;             // 16-byte accesses to them
};

template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const T* p, bool vec) {
  if (vec) {
    const uint4 w4 = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      T e[2];
      *reinterpret_cast<uint32_t*>(e) = w[y];
      x[2 * y] = to_f(e[0]);
      x[2 * y + 1] = to_f(e[1]);
    }
  } else {
#pragma unroll
    for (int y = 0; y < 8; ++y) x[y] = to_f(p[y]);
  }
}

// the row's place: sequence, head, position; false where there is none (padding, or a page that does not exist)
struct Place {
  int b, hk, m, page;
  int64_t token;  // row index into the cache's tensors
};
__device__ __forceinline__ bool find_place(const CacheParams& c, const CacheBatch& bt, int rows, int64_t row, Place* at,
                                           bool* bad) {
  at->m = (int)(row % rows);
  const int64_t bh = row / rows;
  at->hk = (int)(bh % c.Hk);
  at->b = (int)(bh / c.Hk);
  const int len = cached_length(bt, c.page_shift, at->b, bad);
  const int pos = len - rows + at->m;
  at->token = -1;
  if (pos < 0) return false;
  at->page = bt.table[(int64_t)at->b * bt.table_stride + (pos >> c.page_shift)];
  if ((unsigned)at->page >= (unsigned)c.pages) {
    *bad = true;
    return true;
  }
  at->token = (((int64_t)at->page * c.Hk + at->hk) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
  return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(256) cache_write_kernel(CacheParams c, CacheBatch bt, CacheRows r, int* status) {
  constexpr int TPR = D / 8, NG = D >= 32 ? D / 32 : 1, GL = D >= 32 ? 4 : 2;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int w = (int)(idx % TPR);
  const int64_t row = idx / TPR;
  const bool second = blockIdx.y != 0;
  const bool in = row < (int64_t)bt.B * c.Hk * r.rows;
  Place at;
  bool bad = false;
  const bool here = in && find_place(c, bt, r.rows, row, &at, &bad) && at.token >= 0;
  float x[8];
#pragma unroll
  for (int y = 0; y < 8; ++y) x[y] = 0.f;
  if (here)
    load8<T>(x, static_cast<const T*>(second ? r.src[1] : r.src[0]) + at.b * (second ? r.sb[1] : r.sb[0]) +
                    at.hk * (second ? r.sh[1] : r.sh[0]) + (int64_t)at.m * (second ? r.ss[1] : r.ss[0]) + w * 8,
             r.vec != 0);
  // largest magnitude of the group; as integers the magnitudes order as they do, and infinities and NaN come last
  uint32_t top = 0u;
#pragma unroll
  for (int y = 0; y < 8; ++y) top = max(top, __float_as_uint(x[y]) & 0x7fffffffu);
#pragma unroll
  for (int s = 1; s < GL; s <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, s));
  uint32_t sbits;  // bf16
  float inv = 0.f;
  if (top >= 0x7f800000u) sbits = 0xffc0u;
  else {
    const __nv_bfloat16 s = __float2bfloat16_rn(__fdiv_rn(__uint_as_float(top), 7.f));
    sbits = *reinterpret_cast<const uint16_t*>(&s);
    if (sbits < 0x0080u) sbits = 0u;  // below the smallest normal number
    else inv = __fdiv_rn(1.f + 9.5367431640625e-7f, __uint_as_float(sbits << 16));
  }
  uint32_t word = 0u;
#pragma unroll
  for (int y = 0; y < 8; ++y) {
    const int mag = inv == 0.f ? 0 : (int)fmaf(fabsf(x[y]), inv, 0.5f);
    word |= (uint32_t)(8 + (x[y] < 0.f ? -mag : mag)) << (4 * y);
  }
  if (here) {
    if (!second) {
      unsigned char* codes = static_cast<unsigned char*>(c.k_codes) + at.token * (D / 2);
      const int gi = w / 4, t = w % 4;
      if (D >= 32) *reinterpret_cast<uint32_t*>(codes + (t * NG + gi) * 4) = __funnelshift_l(word, word, 2);
      else *reinterpret_cast<uint32_t*>(codes + w * 4) = word;  // half-word t: elements 4 t .. 4 t + 3
    } else {
      unsigned char* codes = static_cast<unsigned char*>(c.v_codes) + at.token * (D / 2);
      const int gi = w / 4, t = w % 4;
      if (D >= 32) {
        word = (word << 2 & 0xfffcfffcu) | (word >> 14 & 0x00030003u);  // each half by itself
        *reinterpret_cast<uint16_t*>(codes + (2 * t * NG + gi) * 2) = (uint16_t)word;
        *reinterpret_cast<uint16_t*>(codes + ((2 * t + 1) * NG + gi) * 2) = (uint16_t)(word >> 16);
      } else {
        *reinterpret_cast<uint32_t*>(codes + w * 4) = word;  // byte g: elements 2 g, 2 g + 1
      }
    }
    if (w % GL == 0)
      static_cast<uint16_t*>(second ? c.v_scales : c.k_scales)[at.token * NG + w / GL] = (uint16_t)sbits;
  }
  if (bad && status != nullptr) atomicOr(status, kBadPage);
}

template <typename T, int D>
__global__ void __launch_bounds__(256) cache_read_kernel(CacheParams c, CacheBatch bt, CacheRows r, int* status) {
  constexpr int TPR = D / 8, NG = D >= 32 ? D / 32 : 1, GL = D >= 32 ? 4 : 2;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int w = (int)(idx % TPR);
  const int64_t row = idx / TPR;
  if (row >= (int64_t)bt.B * c.Hk * r.rows) return;
  const bool second = blockIdx.y != 0;
  Place at;
  bool bad = false;
  const bool real = find_place(c, bt, r.rows, row, &at, &bad);
  uint32_t word = 0x88888888u, sbits = 0u;  // padding: zeros
  if (real && at.token < 0) sbits = 0xffc0u;
  else if (real) {
    sbits = static_cast<const uint16_t*>(second ? c.v_scales : c.k_scales)[at.token * NG + w / GL];
    const int gi = w / 4, t = w % 4;
    if (!second) {
      const unsigned char* codes = static_cast<const unsigned char*>(c.k_codes) + at.token * (D / 2);
      word = *reinterpret_cast<const uint32_t*>(codes + (D >= 32 ? (t * NG + gi) * 4 : w * 4));
      if (D >= 32) word = __funnelshift_r(word, word, 2);
    } else {
      const unsigned char* codes = static_cast<const unsigned char*>(c.v_codes) + at.token * (D / 2);
      if (D >= 32) {
        word = (uint32_t)*reinterpret_cast<const uint16_t*>(codes + (2 * t * NG + gi) * 2) |
               (uint32_t)*reinterpret_cast<const uint16_t*>(codes + ((2 * t + 1) * NG + gi) * 2) << 16;
        word = (word >> 2 & 0x3fff3fffu) | (word << 14 & 0xc000c000u);
      } else word = *reinterpret_cast<const uint32_t*>(codes + w * 4);
    }
  }
  const float s = __uint_as_float(sbits << 16);
  T* dst = static_cast<T*>(second ? r.dst[1] : r.dst[0]) + at.b * (second ? r.sb[1] : r.sb[0]) +
           at.hk * (second ? r.sh[1] : r.sh[0]) + (int64_t)at.m * (second ? r.ss[1] : r.ss[0]) + w * 8;
  uint32_t out[4];
#pragma unroll
  for (int y = 0; y < 4; ++y)
    out[y] = pack2<T>(s * (float)((int)(word >> (8 * y) & 15u) - 8), s * (float)((int)(word >> (8 * y + 4) & 15u) - 8));
  if (r.vec) *reinterpret_cast<uint4*>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
  else {
#pragma unroll
    for (int y = 0; y < 8; ++y) reinterpret_cast<uint16_t*>(dst)[y] = (uint16_t)(out[y / 2] >> (16 * (y & 1)));
  }
  if (bad && status != nullptr) atomicOr(status, kBadPage);
}

// ---------------------------------------------------------------------------------------------- attention
// One kv head's RT rows (the M query rows of each of its G query heads, one head after the other, 8 or 16 at a time)
// against the tokens they see, in tiles of 128.  The bytes of the cache bound it, so the tiles of all sequences and heads
// are one list that is cut into equal shares, a CTA each: lengths are on the device, and no share waits for the longest
// sequence.  What a share has of an item (a row block) that it does not finish goes to the workspace, and a second kernel
// adds up the parts of each item in order.
//   warp 4      brings tiles into shared memory: codes and scales of a page and head are one bulk copy each
//   warps 0-3   take 32 tokens of a tile each, with a running maximum, sum and output of their own, merged at the end
// Matrix instructions are mma.sync m16n8k16 in fp16: a tile has 8 or 16 rows, and the operands come out of registers, where
// a nibble n in bits 2..5 of a half IS the number n 2^-22 (a subnormal): unpacking is one AND per pair, one rotation
// per two.  Nibbles in bits 6..9 are 16 n 2^-22: the query's elements there (the output's rows there) carry 1/16.  The
// matrix instructions align a subnormal as they do 2^-14, so that its products keep 2^-16 of a code, for nibbles in bits 6..9
// 2^-20; with nibbles in bits 0..3 and 4..7 it would be 2^-14 and 2^-18.
//   S = sum_g s_g (sum_d q_d n_d - 8 sum_d q_d)    per group g of the key: the scale multiplies the fp32 product, the sum of
//                                                  q comes in as the accumulator's start.  q is moved by a power of two per
//                                                  row to just below 2^15, so that fp16 holds bf16 queries too.
//   O_d = sum_j (P_j s_jg) n_jd - 8 sum_j P_j s_jg  the scale of the value goes onto the weight; the second sum is one more
//                                                  matrix instruction per group, with the same rounded weights.
// Weights are fp16: 2^-12 of each.  The running maximum is that of S + log2 s, so that P s stays within fp16 for values of
// any size; what falls below 2^-24 of the largest weighted value is lost.
constexpr int TT = 128;       // tokens of a tile
constexpr int STAGES = 4;
constexpr int CONSUMERS = 4;  // warps
constexpr int CTA_THREADS = 32 * (CONSUMERS + 1);
constexpr int CTAS_PER_SM = 2;
constexpr uint32_t kLow = 0x003c003cu, kHigh = 0x03c003c0u;  // the two nibbles of each half's mantissa

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// Tiles that the rows of a sequence see: [0, ns), then [w0, w0 + nt - ns).
struct Span {
  int len, lo, ns, w0, nt;
  __device__ __forceinline__ int tile(int it) const { return it < ns ? it : w0 + it - ns; }
};
__device__ __forceinline__ Span span_of(const CacheAttnParams& p, int b, bool* bad) {
  Span s;
  s.len = cached_length(p.batch, p.cache.page_shift, b, bad);
  s.lo = max(0, s.len - p.M - p.window + 1);  // the first key that the first row's window has
  s.w0 = s.lo / TT;
  s.ns = min((min(p.sinks, s.len) + TT - 1) / TT, s.w0);
  s.nt = s.len > 0 ? s.ns + (s.len + TT - 1) / TT - s.w0 : 0;
  return s;
}

// The tiles of all items (b, kv head, row block) in a row, cut into `shares`.
struct Shares {
  long long total;
  int shares;
  __device__ __forceinline__ long long begin(int c) const { return total * c / shares; }
};
// Warp-wide.  With `find`: the sequence that holds tile `find` of the list, and the list's index of its first tile.
__device__ __forceinline__ long long scan_tiles(const CacheAttnParams& p, int lane, long long find, int* b_found,
                                                long long* b_start) {
  long long base = 0;
  const int per = p.cache.Hk * p.row_blocks;
  bool bad = false;
  for (int b0 = 0; b0 < p.batch.B; b0 += 32) {
    const int b = b0 + lane;
    long long n = b < p.batch.B ? (long long)span_of(p, b, &bad).nt * per : 0;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, n, s);
      if (lane >= s) n += up;
    }
    if (find >= 0) {
      const unsigned past = __ballot_sync(0xffffffffu, base + n > find);
      if (past != 0u) {
        const int first = __ffs(past) - 1;
        const long long before = __shfl_up_sync(0xffffffffu, n, 1);
        *b_start = base + (first == 0 ? 0 : __shfl_sync(0xffffffffu, before, first));
        *b_found = b0 + first;
        return -1;
      }
    }
    base += __shfl_sync(0xffffffffu, n, 31);
  }
  if (bad && p.status != nullptr) atomicOr(p.status, kBadPage);
  return base;
}
__device__ __forceinline__ Shares make_shares(const CacheAttnParams& p, long long total) {
  const long long most = (total + p.min_tiles - 1) / p.min_tiles;
  return {total, (int)max(1ll, min((long long)p.grid, most))};
}

// A share's walk over its segments, each some tiles of one item.
struct Walk {
  long long at, end;  // in the list of tiles
  int b, item;        // item: kv head * row_blocks + row block
  int first;          // first tile of the segment within its item
  Span span;
  __device__ __forceinline__ int count() const { return (int)min((long long)(span.nt - first), end - at); }
};
__device__ __forceinline__ bool walk_begin(const CacheAttnParams& p, int lane, Walk* w) {
  const Shares sh = make_shares(p, scan_tiles(p, lane, -1, nullptr, nullptr));
  if ((int)blockIdx.x >= sh.shares) return false;
  w->at = sh.begin(blockIdx.x);
  w->end = sh.begin(blockIdx.x + 1);
  if (w->at >= w->end) return false;
  long long start = 0;
  scan_tiles(p, lane, w->at, &w->b, &start);
  bool bad = false;
  w->span = span_of(p, w->b, &bad);
  const long long off = w->at - start;
  w->item = (int)(off / w->span.nt);
  w->first = (int)(off % w->span.nt);
  return true;
}
__device__ __forceinline__ bool walk_next(const CacheAttnParams& p, Walk* w) {
  w->at += w->count();
  if (w->at >= w->end) return false;
  w->first = 0;
  if (++w->item >= p.cache.Hk * p.row_blocks) {
    w->item = 0;
    bool bad = false;
    do {
      ++w->b;
      w->span = span_of(p, w->b, &bad);
    } while (w->span.nt == 0);  // (the list has more tiles, so a later sequence has some)
  }
  return true;
}

template <int D, int RT>
struct CacheSmem {
  static constexpr int NG = D >= 32 ? D / 32 : 1;
  static constexpr int kRow = D / 2, kScale = NG * 2;  // bytes of a token
  static constexpr int k_off = 0, v_off = TT * kRow, ks_off = 2 * TT * kRow, vs_off = ks_off + TT * kScale;
  static constexpr int kStage = vs_off + TT * kScale;
  static constexpr int out_off = STAGES * kStage;  // CONSUMERS x RT x (D + 4) floats, then (m, l) of them
  static constexpr int kOutRow = D + 4;
  static constexpr int ml_off = out_off + CONSUMERS * RT * kOutRow * 4;
  static constexpr int bar_off = ml_off + CONSUMERS * RT * 8;
  static constexpr int total = bar_off + 128;
};
struct CacheBars {
  uint64_t full[STAGES], empty[STAGES];
  int abort_flag;
};
static_assert(sizeof(CacheBars) <= 128, "room for the barriers");

// Workspace: per share two slots of RT rows: D floats, then the row's maximum (log2 units) and sum.
// Slot 0: the share's first segment, where it does not begin its item; slot 1: the last, where it begins its item but does not end it.
template <int D, int RT>
__device__ __forceinline__ float* part_slot(float* ws, int share, int slot) {
  return ws + ((int64_t)share * 2 + slot) * RT * (D + 2);
}

// Four elements of a finished row: sum / den, zeros for a row that saw nothing.
template <typename T>
__device__ __forceinline__ void store_row(const CacheAttnParams& p, int b, int hk, int r, int d, float4 sum, float top, float den) {
  if (r >= p.rows) return;
  const int head = hk * p.G + r / p.M, i = r % p.M;
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

template <typename T, int D, int RT>
__global__ void __launch_bounds__(CTA_THREADS, CTAS_PER_SM) cache_attn_kernel(const CacheAttnParams p) {
  using L = CacheSmem<D, RT>;
  constexpr int NG = L::NG;
  constexpr int MT = D >= 32 ? 2 : 1;  // 16-row tiles of a group's output
  constexpr int NB = RT / 8;           // blocks of 8 rows
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
  Walk w;
  const bool any = walk_begin(p, lane, &w);  // (the same in every warp)

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
    int n = 0;  // tiles so far
    bool ok = true, bad = false;
    do {
      const int hk = w.item / p.row_blocks, cnt = w.count();
      for (int it = 0; ok && it < cnt; ++it, ++n) {
        const int t0 = w.span.tile(w.first + it) * TT;
        // what may be seen of the tile: the sinks, the windows, or both
        int lo = max(t0, w.span.lo), hi = min(t0 + TT, w.span.len);
        if (t0 < p.sinks) {
          if (lo >= hi) hi = min(hi, p.sinks);
          lo = t0;
        }
        const int p0 = t0 + (piece << shift);
        lo = max(lo, p0) & ~15;
        hi = min((min(hi, p0 + (1 << shift)) + 15) & ~15, p0 + (1 << shift));
        const int s = n % STAGES;
        unsigned char* stage = smem + s * L::kStage;
        int page = -1;
        const bool copy = mine && lo < hi;
        if (copy) page = p.batch.table[(int64_t)w.b * p.batch.table_stride + (p0 >> p.cache.page_shift)];
        ok = mbar_wait(&bars->empty[s], ((n / STAGES) & 1) ^ 1, abort_flag);
        if (!ok) break;
        unsigned char* dst = stage + off + (lo - t0) * bytes;
        const int size = (hi - lo) * bytes;
        if (copy && (unsigned)page < (unsigned)p.cache.pages) {
          mbar_arrive_expect_tx(&bars->full[s], size);
          const int64_t row = (((int64_t)page * p.cache.Hk + hk) << p.cache.page_shift) + (lo & ((1 << p.cache.page_shift) - 1));
          bulk_load_1d(dst, src + row * bytes, size, &bars->full[s]);
        } else {
          if (copy) {  // a page that does not exist: its keys are NaN
            bad = true;
            if (kind == 2) {
              for (int x = 0; x < size; x += 4) *reinterpret_cast<uint32_t*>(dst + x) = 0xffc0ffc0u;
              fence_proxy_async_smem();  // (later copies go over them)
            }
          }
          mbar_arrive(&bars->full[s]);
        }
      }
    } while (ok && walk_next(p, &w));
    if (bad && p.status != nullptr) atomicOr(p.status, kBadPage);
  } else if (any) {
    // ------------------------------------------------------------ rows
    const int g = lane >> 2, t = lane & 3;
    // tokens of this lane's four columns of 16, and the key row that it loads for each block of eight columns
    const int tok[4] = {t, (t ^ 1) + 4, t + 8, (t ^ 1) + 12};
    const int krow = (g & 1) ? ((g >> 1) ^ 1) + 4 : g >> 1;
    float* so = reinterpret_cast<float*>(smem + L::out_off) + warp * RT * L::kOutRow;
    float2* ml = reinterpret_cast<float2*>(smem + L::ml_off);
    int n = 0;
    bool ok = true;
    do {
      const int hk = w.item / p.row_blocks, r0 = (w.item % p.row_blocks) * RT, cnt = w.count();
      // ---- the rows' queries as fp16 operands, and -8 sum of each group
      uint32_t q[NG][2][4];
      float qbias[NB][NG], f[NB];
      int hi_row[NB], lo_row[NB];  // a row sees keys [lo_row, hi_row) and the sinks before hi_row
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int r = r0 + nb * 8 + g;
        const bool real = r < p.rows;
        const int head = r / p.M, i = r - head * p.M;
        hi_row[nb] = real ? w.span.len - p.M + i + 1 : 0;
        lo_row[nb] = hi_row[nb] - p.window;
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
        f[nb] = p.sm_scale * kLog2e * __int_as_float((127 + 22) << 23) * __int_as_float((127 - k) << 23);
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
          qbias[nb][gi] = -8.f * 2.384185791015625e-7f * sum;
          auto pair = [&](int a, int b) {
            return (uint32_t)__half_as_ushort(h[a]) | (uint32_t)__half_as_ushort(h[b]) << 16;
          };
          // element y of a word is nibble y: registers (0, 4), (1, 5), (2, 6), (3, 7)
          q[gi][0][nb] = pair(0, 4);
          q[gi][0][2 + nb] = pair(1, 5);
          q[gi][1][nb] = pair(2, 6);
          q[gi][1][2 + nb] = pair(3, 7);
          if (NB == 1) q[gi][0][1] = q[gi][0][3] = q[gi][1][1] = q[gi][1][3] = 0u;
        }
      }
      float o[NB][NG][MT][4], ob[NB][NG][4], m[NB], l[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        m[nb] = FAWS_NEG_INF;
        l[nb] = 0.f;
#pragma unroll
        for (int gi = 0; gi < NG; ++gi)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            ob[nb][gi][c] = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) o[nb][gi][mt][c] = 0.f;
          }
      }
      const int hi_first = w.span.len - p.M + 1, lo_last = w.span.len - p.window;  // of the first, the last row

      // ---- 16 tokens from `base` of the stage on, the first of them at position n0
      auto step = [&](auto masked_tag, const unsigned char* stage, int base, int n0) {
        constexpr bool kMasked = decltype(masked_tag)::value;
        float s[NB][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const unsigned char* kr = stage + L::k_off + (base + half * 8 + krow) * L::kRow;
          uint32_t kw[NG];
          if constexpr (NG == 4) *reinterpret_cast<uint4*>(kw) = *reinterpret_cast<const uint4*>(kr + t * 16);
          else if constexpr (NG == 2) *reinterpret_cast<uint2*>(kw) = *reinterpret_cast<const uint2*>(kr + t * 8);
          else if constexpr (D == 32) kw[0] = *reinterpret_cast<const uint32_t*>(kr + t * 4);
          else kw[0] = (uint32_t)*reinterpret_cast<const uint16_t*>(kr + t * 2) << 2;  // elements 4 t .. + 3, then none
          float acc[NG][4];
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            acc[gi][0] = acc[gi][1] = qbias[0][gi];
            acc[gi][2] = acc[gi][3] = NB == 2 ? qbias[NB - 1][gi] : 0.f;
            const uint32_t lo = kw[gi], hi = __funnelshift_r(kw[gi], kw[gi], 8);
            mma_f16(acc[gi], q[gi][0], lo & kLow, lo & kHigh);
            mma_f16(acc[gi], q[gi][1], hi & kLow, hi & kHigh);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const unsigned char* sp = stage + L::ks_off + (base + tok[half * 2 + e]) * L::kScale;
            float sc[NG];
            if constexpr (NG == 4) {
              const uint2 w2 = *reinterpret_cast<const uint2*>(sp);
              sc[0] = bf16_lo(w2.x); sc[1] = bf16_hi(w2.x); sc[2] = bf16_lo(w2.y); sc[3] = bf16_hi(w2.y);
            } else if constexpr (NG == 2) {
              const uint32_t w1 = *reinterpret_cast<const uint32_t*>(sp);
              sc[0] = bf16_lo(w1); sc[1] = bf16_hi(w1);
            } else sc[0] = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(sp) << 16);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              float x = sc[0] * acc[0][nb * 2 + e];
#pragma unroll
              for (int gi = 1; gi < NG; ++gi) x = fmaf(sc[gi], acc[gi][nb * 2 + e], x);
              s[nb][half * 2 + e] = x * f[nb];
            }
          }
        }
        if constexpr (kMasked) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = n0 + tok[e];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              if (!(j < hi_row[nb] && (j >= lo_row[nb] || j < p.sinks))) s[nb][e] = FAWS_NEG_INF;
          }
        }
        // ---- value scales, and about log2 of the largest of each token
        float vs[4][NG], ev[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned char* sp = stage + L::vs_off + (base + tok[e]) * L::kScale;
          int top;
          if constexpr (NG == 4) {
            const uint2 w2 = *reinterpret_cast<const uint2*>(sp);
            vs[e][0] = bf16_lo(w2.x); vs[e][1] = bf16_hi(w2.x); vs[e][2] = bf16_lo(w2.y); vs[e][3] = bf16_hi(w2.y);
            const uint32_t mx = __vmaxs2(w2.x, w2.y);
            top = max((int)(mx << 16), (int)(mx & 0xffff0000u));
          } else if constexpr (NG == 2) {
            const uint32_t w1 = *reinterpret_cast<const uint32_t*>(sp);
            vs[e][0] = bf16_lo(w1); vs[e][1] = bf16_hi(w1);
            top = max((int)(w1 << 16), (int)(w1 & 0xffff0000u));
          } else {
            top = (int)((uint32_t)*reinterpret_cast<const uint16_t*>(sp) << 16);
            vs[e][0] = __int_as_float(top);
          }
          // exponent and fraction of a float, read as an integer, are its log2 to 0.09; a NaN (negative) has none
          ev[e] = fmaxf((float)top * 1.1920928955078125e-7f - 127.f, -100.f);
        }
        // ---- running maximum, moved only when a weighted value would exceed 2^8
        bool need = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float mx = s[nb][0] + ev[0];
#pragma unroll
          for (int e = 1; e < 4; ++e) mx = fmaxf(mx, s[nb][e] + ev[e]);
          need = need || mx > m[nb] + 8.f;
        }
        if (__any_sync(0xffffffffu, need)) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float mx = s[nb][0] + ev[0];
#pragma unroll
            for (int e = 1; e < 4; ++e) mx = fmaxf(mx, s[nb][e] + ev[e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m[nb], mx);
            const float alpha = m_new == FAWS_NEG_INF ? 1.f : fast_exp2(m[nb] - m_new);
            m[nb] = m_new;
            l[nb] *= alpha;
            // the outputs' columns 2 t and 2 t + 1 are rows of other lanes
            const float a0 = __shfl_sync(0xffffffffu, alpha, t * 8), a1 = __shfl_sync(0xffffffffu, alpha, t * 8 + 4);
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
              ob[nb][gi][0] *= a0; ob[nb][gi][1] *= a1; ob[nb][gi][2] *= a0; ob[nb][gi][3] *= a1;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                o[nb][gi][mt][0] *= a0; o[nb][gi][mt][1] *= a1; o[nb][gi][mt][2] *= a0; o[nb][gi][mt][3] *= a1;
              }
            }
          }
        }
        float pr[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const float ms = m[nb] == FAWS_NEG_INF ? 0.f : m[nb];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pr[nb][e] = fast_exp2(s[nb][e] - ms);
            l[nb] += pr[nb][e];
          }
        }
        // ---- values
        uint32_t vw[4][(NG + 1) / 2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned char* vr = stage + L::v_off + (base + tok[e]) * L::kRow;
          if constexpr (NG == 4) *reinterpret_cast<uint2*>(vw[e]) = *reinterpret_cast<const uint2*>(vr + g * 8);
          else if constexpr (NG == 2) vw[e][0] = *reinterpret_cast<const uint32_t*>(vr + g * 4);
          else if constexpr (D == 32) vw[e][0] = *reinterpret_cast<const uint16_t*>(vr + g * 2);
          else vw[e][0] = vr[g];
        }
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          // both tokens' half-words of the group; then with their bytes exchanged, which brings the next two nibbles
          const uint32_t sel = (gi & 1) ? 0x7632u : 0x5410u, swapped = (gi & 1) ? 0x6723u : 0x4501u;
          uint32_t x01 = __byte_perm(vw[0][gi >> 1], vw[1][gi >> 1], sel), x23 = __byte_perm(vw[2][gi >> 1], vw[3][gi >> 1], sel);
          if (D == 16) {
            x01 <<= 2;
            x23 <<= 2;
          }
          const uint32_t a0[4] = {x01 & kLow, x01 & kHigh, x23 & kLow, x23 & kHigh};
          const uint32_t ab[4] = {0x00200020u, 0x02000200u, 0x00200020u, 0x02000200u};  // 8 in every place
          [[maybe_unused]] uint32_t a1[4];
          if constexpr (MT == 2) {
            const uint32_t y01 = __byte_perm(vw[0][gi >> 1], vw[1][gi >> 1], swapped);
            const uint32_t y23 = __byte_perm(vw[2][gi >> 1], vw[3][gi >> 1], swapped);
            a1[0] = y01 & kLow; a1[1] = y01 & kHigh; a1[2] = y23 & kLow; a1[3] = y23 & kHigh;
          }
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float pv[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              pv[e] = pr[nb][e] * vs[e][gi];
              if (kMasked && pr[nb][e] == 0.f) pv[e] = 0.f;  // a hidden token's scale may be anything
            }
            const uint32_t b0 = pack2<__half>(pv[0], pv[1]), b1 = pack2<__half>(pv[2], pv[3]);
            mma_f16(o[nb][gi][0], a0, b0, b1);
            if constexpr (MT == 2) mma_f16(o[nb][gi][MT - 1], a1, b0, b1);
            mma_f16(ob[nb][gi], ab, b0, b1);
          }
        }
      };

      for (int it = 0; ok && it < cnt; ++it, ++n) {
        const int t0 = w.span.tile(w.first + it) * TT, st = n % STAGES;
        ok = mbar_wait(&bars->full[st], (n / STAGES) & 1, abort_flag);
        if (!ok) break;
        const unsigned char* stage = smem + st * L::kStage;
        const int n0 = t0 + warp * 32;
        const bool whole = n0 + 32 <= hi_first && (n0 >= lo_last || n0 + 32 <= p.sinks);
        // (32 tokens that no row sees are skipped)
        if (whole) {
          step(std::false_type{}, stage, warp * 32, n0);
          step(std::false_type{}, stage, warp * 32 + 16, n0 + 16);
        } else {
#pragma unroll 1
          for (int x = 0; x < 32; x += 16)
            if (n0 + x < w.span.len && (n0 + x + 16 > w.span.lo || n0 + x < p.sinks))
              step(std::true_type{}, stage, warp * 32 + x, n0 + x);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->empty[st]);
      }

      // ---- the four warps' parts
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float ls = l[nb];
        ls += __shfl_xor_sync(0xffffffffu, ls, 1);
        ls += __shfl_xor_sync(0xffffffffu, ls, 2);
        if (t == 0) ml[warp * RT + nb * 8 + g] = make_float2(m[nb], ls);
#pragma unroll
        for (int gi = 0; gi < NG; ++gi)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int row = nb * 8 + 2 * t + (c & 1);
              const int d = D >= 32 ? 32 * gi + 4 * g + 2 * mt + (c >> 1) : 2 * g + (c >> 1);
              so[row * L::kOutRow + d] = (o[nb][gi][mt][c] - ob[nb][gi][c]) * (c >> 1 ? 262144.f : 4194304.f);
            }
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
          store_row<T>(p, w.b, hk, r0 + row, d, sum, top, den);
        } else {
          float* part = part_slot<D, RT>(p.parts, blockIdx.x, begins ? 1 : 0) + row * (D + 2);
          part[d] = sum.x; part[d + 1] = sum.y; part[d + 2] = sum.z; part[d + 3] = sum.w;
          if (d == 0) { part[D] = top; part[D + 1] = den; }
        }
      }
      ok = !consumers_any(!ok);  // (all of them go on, or none)
    } while (ok && walk_next(p, &w));
  }
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, 1);
    for (int x = 0; x < 50; ++x) __nanosleep(20000);  // let copies in flight land before the smem goes away
    __syncthreads();
  }
}

// The parts of the items that several shares had, added up in the order of the shares; zeros where a row block saw nothing.
// A CTA per item.
template <typename T, int D, int RT>
__global__ void __launch_bounds__(128) cache_combine_kernel(const CacheAttnParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int items = p.cache.Hk * p.row_blocks;
  const int b = (int)(blockIdx.x / (unsigned)items), item = (int)(blockIdx.x % (unsigned)items);
  const int hk = item / p.row_blocks, r0 = (item % p.row_blocks) * RT;
  bool bad = false;
  const Span span = span_of(p, b, &bad);
  if (span.nt == 0) {
    for (int x = threadIdx.x; x < RT * (D / 4); x += 128)
      store_row<T>(p, b, hk, r0 + x / (D / 4), (x % (D / 4)) * 4, make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f);
    return;
  }
  // tiles of the list before this item, and in all
  long long before = 0, total = 0;
  for (int b0 = 0; b0 < p.batch.B; b0 += 32) {
    const long long n = b0 + lane < p.batch.B ? (long long)span_of(p, b0 + lane, &bad).nt * items : 0;
    long long all = n, less = b0 + lane < b ? n : 0;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, s);
      less += __shfl_xor_sync(0xffffffffu, less, s);
    }
    total += all;
    before += less;
  }
  before += (long long)item * span.nt;
  const Shares sh = make_shares(p, total);
  auto share_of = [&](long long tile) {  // the share that has it
    int c = (int)(((tile + 1) * sh.shares - 1) / total);
    while (sh.begin(c + 1) <= tile) ++c;
    while (sh.begin(c) > tile) --c;
    return c;
  };
  const int c0 = share_of(before), c1 = share_of(before + span.nt - 1);
  if (c0 == c1) return;  // one share had all of it
  for (int x = threadIdx.x; x < RT * (D / 4); x += 128) {
    const int row = x / (D / 4), d = (x % (D / 4)) * 4;
    float top = FAWS_NEG_INF;
    for (int c = c0; c <= c1; ++c) top = fmaxf(top, part_slot<D, RT>(p.parts, c, c == c0 ? 1 : 0)[row * (D + 2) + D]);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
    for (int c = c0; c <= c1; ++c) {
      const float* part = part_slot<D, RT>(p.parts, c, c == c0 ? 1 : 0) + row * (D + 2);
      const float e = part[D] == FAWS_NEG_INF ? 0.f : fast_exp2(part[D] - top);
      den = fmaf(e, part[D + 1], den);
      sum.x = fmaf(e, part[d], sum.x); sum.y = fmaf(e, part[d + 1], sum.y);
      sum.z = fmaf(e, part[d + 2], sum.z); sum.w = fmaf(e, part[d + 3], sum.w);
    }
    store_row<T>(p, b, hk, r0 + row, d, sum, top, den);
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

template <typename T, int D, int RT>
cudaError_t launch_attn_r(CacheAttnParams p, cudaStream_t s) {
  using L = CacheSmem<D, RT>;
  static PerDeviceOnce once;
  if (cudaError_t e = set_max_smem_once(once, cache_attn_kernel<T, D, RT>, L::total); e != cudaSuccess) return e;
  p.row_blocks = (p.rows + RT - 1) / RT;
  if (cudaError_t e = launch_overlapped(cache_attn_kernel<T, D, RT>, dim3(p.grid), CTA_THREADS, L::total, s, p); e != cudaSuccess)
    return e;
  const unsigned items = (unsigned)(p.batch.B * p.cache.Hk * p.row_blocks);
  return launch_overlapped(cache_combine_kernel<T, D, RT>, dim3(items), 128, 0, s, p);
}
template <typename T, int D>
cudaError_t launch_attn_d(const CacheAttnParams& p, cudaStream_t s) {
  return p.rows <= 8 ? launch_attn_r<T, D, 8>(p, s) : launch_attn_r<T, D, 16>(p, s);
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

template <typename T, bool WRITE>
cudaError_t launch_rows_t(const CacheParams& c, const CacheBatch& b, const CacheRows& r, cudaStream_t s) {
  const int64_t threads = (int64_t)b.B * c.Hk * r.rows * (c.D / 8);
  const dim3 grid((unsigned)((threads + 255) / 256), 2, 1);
  int* status = tc_status_word();
#define FAWS_ROWS(D)                                                                          \
  return launch_overlapped(WRITE ? cache_write_kernel<T, D> : cache_read_kernel<T, D>, grid, 256, 0, s, c, b, r, status)
  switch (c.D) {
    case 16: FAWS_ROWS(16);
    case 32: FAWS_ROWS(32);
    case 64: FAWS_ROWS(64);
    default: FAWS_ROWS(128);
  }
#undef FAWS_ROWS
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

size_t cache_attn_workspace_bytes(int rows, int D) {
  return (size_t)shares_at_most() * 2 * (rows <= 8 ? 8 : 16) * (D + 2) * 4;
}

cudaError_t launch_cache_attn(const CacheAttnParams& call, int dtype, cudaStream_t s) {
  CacheAttnParams p = call;
  p.grid = shares_at_most();
  p.min_tiles = 2;
  p.vec_out = reinterpret_cast<uintptr_t>(p.out) % 8 == 0 && p.o_sb % 4 == 0 && p.o_sh % 4 == 0 && p.o_ss % 4 == 0;
  p.status = tc_status_word();
  return dtype == FAWS_FP16 ? launch_attn_t<__half>(p, s) : launch_attn_t<__nv_bfloat16>(p, s);
}

}  // namespace faws
