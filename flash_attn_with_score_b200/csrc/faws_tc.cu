// tcgen05 / TMEM / TMA kernels (sm_100a) of the attention-with-scores family: the forward launches (kernel in
// faws_tc_fwd.cuh), the key-major pass of the softmax sums, and the status word of bounded waits.
#include <cuda.h>

#include <cstdio>
#include <cstdlib>
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "faws_tc_fwd.cuh"

namespace faws {
namespace {
using namespace ptx;

// ---------------------------------------------------------------------------- key-major pass
// Softmax column sums from a saved log-normaliser (the structure of total.py:50-142 and of the
// reference's second passes, attention_with_col_softmax_sum.py:195-270,
// attention_cross_token_softmax_sum.py:203-268, without atomics):
//   out[j] = sum over heads of the CTA and queries i of exp(s_ij - L_i).
// One CTA owns 128 keys of one (batch, kv head or query head) and walks the query tiles of its
// heads.  S^T = K.Q^T puts keys on TMEM lanes, so thread j accumulates column j in a register:
// no cross-thread reduction, fixed order, one store.
// One CTA owns CS_KT = 2 key tiles (256 keys) of one (batch, kv head or query head): every Q tile
// it streams feeds two MMAs, which halves the Q traffic from L2 (32 KB per 128^3 MMA otherwise).
// (Measured: 1-3 % faster, not more: halving the Q traffic, and, in a separate experiment, moving half of
// the exponentials from the MUFU pipe to a cubic on the FMA pipe, both left the pass where it was.)
// Four consumer warpgroups: warpgroup w owns S^T buffer w = key tile (w & 1) of the query tiles
// of parity (w >> 1); it walks its tiles in chunks of CS_CHUNK columns (that many live score
// registers); the two partial sums of a key tile are added in a fixed order at the end.
constexpr int CS_KT = 2;
constexpr int CS_WGS = 4;
constexpr int CS_QSLOTS = CS_WGS;
constexpr int CS_CHUNK = 64;  // score columns a consumer thread holds at a time
constexpr int CS_LSLOTS = 8;  // query tiles whose -L values are in shared memory (see the producer)
constexpr int CS_THREADS = 128 + CS_WGS * 128;
constexpr int CS_REGS_LAUNCH = (65536 / CS_THREADS) & ~7;  // what the launch bound lets ptxas allocate
constexpr int CS_REGS_AUX = 56;
constexpr int CS_REGS_CONSUMER = ((CS_REGS_LAUNCH * CS_THREADS - 128 * CS_REGS_AUX) / (CS_WGS * 128)) & ~7;
static_assert(128 * CS_REGS_AUX + CS_WGS * 128 * CS_REGS_CONSUMER <= CS_REGS_LAUNCH * CS_THREADS,
              "setmaxnreg would block");
static_assert(CS_WGS == 2 * CS_KT, "buffer w = key tile (w & 1) of query-tile parity (w >> 1)");

template <int D>
struct CsSmem {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kSub = 128 * 128;
  static constexpr int k_off = 0;                           // CS_KT key tiles
  static constexpr int q_off = k_off + CS_KT * kTile;
  static constexpr int l_off = q_off + CS_QSLOTS * kTile;  // [warpgroup][2][128] floats: -L_i*log2e per query
  static constexpr int comb_off = l_off + CS_WGS * 2 * 128 * 4;  // [key tile][128] floats
  static constexpr int bar_off = comb_off + CS_KT * 128 * 4;
  static constexpr int total = bar_off + 256;
  static constexpr int alloc = total + 1024;
};

struct CsBars {
  uint64_t k_full;
  uint64_t q_full[CS_QSLOTS], q_empty[CS_QSLOTS];
  uint64_t s_full[CS_WGS], s_free[CS_WGS];  // per S^T buffer
  uint64_t l_ready[CS_WGS];
  uint64_t l_full[CS_LSLOTS];  // -L*log2e of a query tile has landed (bulk copy from the padded array)
  uint32_t tmem_base;
  int abort_flag;
};

struct CsMaps {
  CUtensorMap q, k;
};

template <typename T, int D>
__global__ void __launch_bounds__(CS_THREADS, 1)
tc_colsoftmax_kernel(const __grid_constant__ CsMaps maps, const ColSoftmaxParams p, int heads_per_cta,
                     int* __restrict__ status) {
  using L = CsSmem<D>;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  CsBars* bars = reinterpret_cast<CsBars*>(smem + L::bar_off);
  volatile int* abort_flag = &bars->abort_flag;
  float* lbuf = reinterpret_cast<float*>(smem + L::l_off);
  float* comb = reinterpret_cast<float*>(smem + L::comb_off);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Causal: key tiles are the slowest grid dimension, so the key tiles that see the most queries
  // (the first ones) of all heads are dispatched first.  Otherwise key tiles are fastest.
  const int n0 = (p.causal ? blockIdx.z : blockIdx.x) * (CS_KT * BN);  // first key of the CTA's CS_KT key tiles
  const int ho = p.causal ? blockIdx.x : blockIdx.y;
  const int b = p.causal ? blockIdx.y : blockIdx.z;
  const int n_heads_out = p.causal ? gridDim.x : gridDim.y;
  const int h0 = ho * heads_per_cta;  // first query head of this CTA
  const int hk = h0 / p.G;

  // query tiles (absolute multiples of 128) the CTA's first key tile needs, per head (the second key tile
  // sees a suffix of them; what it does not see is masked)
  const int i_lo = max(p.i_begin, p.m_begin);
  int i_first = i_lo;
  if (p.causal) i_first = max(i_first, n0 - p.p_seq);
  const int qt0 = i_first / BM;
  const int ntq = max(0, (p.m_end + BM - 1) / BM - qt0);
  const int total = ntq * heads_per_cta;

  if (threadIdx.x == 0) {
    mbar_init(&bars->k_full, 1);
    for (int s = 0; s < CS_QSLOTS; ++s) {
      mbar_init(&bars->q_full[s], 1);
      mbar_init(&bars->q_empty[s], 1);
    }
    for (int w = 0; w < CS_WGS; ++w) {
      mbar_init(&bars->s_full[w], 1);
      mbar_init(&bars->s_free[w], 128);
      mbar_init(&bars->l_ready[w], 128);
    }
    for (int l = 0; l < CS_LSLOTS; ++l) mbar_init(&bars->l_full[l], 1);
    bars->abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&maps.q);
    prefetch_tmap(&maps.k);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;

  float acc = 0.f;
  if (warp < 4) {
    reg_dealloc<CS_REGS_AUX>();
    if (warp == 0 && lane == 0 && total > 0) {
      // ---------------------------------------------------------- TMA producer
      mbar_arrive_expect_tx(&bars->k_full, CS_KT * L::kTile);
      for (int kt = 0; kt < CS_KT; ++kt)
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(smem + L::k_off + kt * L::kTile + c * L::kSub, &maps.k, &bars->k_full, c * 64, n0 + kt * BN, hk, b);
      // -L_i*log2e of query tile u goes to slot u % 8 by one 512-byte bulk copy, issued after the Q load
      // of tile u.  That load waited for the MMA of tile u - 4, which was issued only after both
      // warpgroups of this parity had taken all of S^T of tile u - 6 out of TMEM, i.e. after they had
      // finished tile u - 8: its slot is free.  The first copy waits for the kernel that wrote the
      // array; the first Q loads (inputs of the whole call) are in flight by then.
      int l_next = 0;
      bool waited = false;
      for (int u = 0; u < total; ++u) {
        const int s = u % CS_QSLOTS, use = u / CS_QSLOTS;
        const int g = u / ntq, qt = qt0 + (u - g * ntq);
        if (!mbar_wait(&bars->q_empty[s], (use & 1) ^ 1, abort_flag)) break;
        mbar_arrive_expect_tx(&bars->q_full[s], L::kTile);
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(smem + L::q_off + s * L::kTile + c * L::kSub, &maps.q, &bars->q_full[s], c * 64, qt * BM,
                      h0 + g, b);
        if (p.negl_pad != nullptr && (u >= CS_QSLOTS - 1 || u == total - 1)) {
          if (!waited) {
            griddep_wait();
            waited = true;
          }
          for (; l_next <= u; ++l_next) {
            const int gl = l_next / ntq, ql = qt0 + (l_next - gl * ntq);
            const int sl = l_next % CS_LSLOTS;
            mbar_arrive_expect_tx(&bars->l_full[sl], BM * 4);
            bulk_load_1d(lbuf + sl * BM, p.negl_pad + ((int64_t)b * p.Hq + h0 + gl) * p.m_pad + ql * BM, BM * 4,
                         &bars->l_full[sl]);
          }
        }
      }
    } else if (warp == 1 && total > 0 && elect_one()) {
      // ---------------------------------------------------------- MMA issuer: S^T = K . Q^T
      // One thread runs this loop: the tensor pipe's queue holds about six 64-cycle MMAs, so that what comes between two
      // groups of them counts once the queue is short.  With the whole warp in the loop and a lane elected for each group
      // (which the forward kernel does as fast either way) bf16 B8 Hq32 Hk32 S1024 D128 causal took 204 us with its forward
      // pass, 199 this way; where the power cap sets the pace (B4 Hq32 Hk8 S16384 full) 26.3 and 26.4 ms.
      constexpr int kFmt = std::is_same<T, __half>::value ? 0 : 1;
      constexpr uint32_t idesc = make_idesc_f16(128, BM, kFmt, 0, 0);
      const int k_steps = D == 64 ? (p.D + 15) / 16 : D / 16;  // (head dims 16 and 32: no K-steps of padding)
      const uint64_t k_desc = make_desc_sw128(smem_u32(smem + L::k_off), 16, 1024);
      const uint64_t q_desc0 = make_desc_sw128(smem_u32(smem + L::q_off), 16, 1024);
      bool ok = mbar_wait(&bars->k_full, 0, abort_flag);
      for (int u = 0; ok && u < total; ++u) {
        const int s = u % CS_QSLOTS, use = u / CS_QSLOTS;
        const int buf0 = (u & 1) * CS_KT, buse = u >> 1;  // S^T buffers of this query tile, and their use count
        if (!(ok = mbar_wait(&bars->q_full[s], use & 1, abort_flag))) break;
        for (int kt = 0; ok && kt < CS_KT; ++kt) ok = mbar_wait(&bars->s_free[buf0 + kt], (buse & 1) ^ 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint64_t qd = q_desc0 + (uint64_t)(s * (L::kTile >> 4));
#pragma unroll
        for (int kt = 0; kt < CS_KT; ++kt) {
          const uint32_t d_tmem = tmem_base + (uint32_t)((buf0 + kt) * BM);
          const uint64_t kd = k_desc + (uint64_t)(kt * (L::kTile >> 4));
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t off = (uint64_t)(((kk >> 2) * L::kSub + (kk & 3) * 32) >> 4);
            if (kk == 0) mma_ss(d_tmem, kd + off, qd + off, idesc, 0u);
            else if (kk < k_steps) mma_ss_acc(d_tmem, kd + off, qd + off, idesc);
          }
          if (kt == CS_KT - 1) mma_commit(&bars->q_empty[s]);
          mma_commit(&bars->s_full[buf0 + kt]);
        }
      }
    }
  } else {
    reg_alloc<CS_REGS_CONSUMER>();
    // ------------------------------------------------------------ consumers: thread = key
    // L comes from the forward pass this launch may overlap (programmatic dependent launch): the
    // consumers are the only threads that read it, and the only ones that write the result.
    griddep_wait();
    const int wg = (warp - 4) >> 2;
    const int lg = warp & 3;
    const int row = lg * 32 + lane;
    const int kt = wg & (CS_KT - 1), par = wg / CS_KT;  // this warpgroup's key tile and query-tile parity
    const int nk0 = n0 + kt * BN;                      // first key of that tile
    const int j = nk0 + row;
    const uint32_t t_buf = tmem_base + ((uint32_t)(lg * 32) << 16) + (uint32_t)(wg * BM);
    const float scale_log2 = p.sm_scale * kLog2e;

    // -L_i*log2e of query tile u (for this thread's column x = row), -inf where the query is
    // outside the summed range or has no visible key
    auto load_negl = [&](int u) -> float {
      const int g = u / ntq, qt = qt0 + (u - g * ntq);
      const int i = qt * BM + row;
      float v = FAWS_NEG_INF;
      if (i >= i_lo && i < p.m_end) {
        const float Li = p.L[((int64_t)b * p.Hq + h0 + g) * p.M + i];
        if (Li != FAWS_NEG_INF) v = -Li * kLog2e;
      }
      return v;
    };

    // A warp without a key of the sum hands its scores back unread (fp16 B16 H8 S785 D32, where that is 7 of a head's 32
    // groups of keys, and one of its 14 half tiles of queries is left out below: 114 -> 108 us with the forward pass).
    const bool no_keys = nk0 + lg * 32 >= p.n_end;
    bool alive = true;
    int mine = 0;  // tiles this warpgroup has processed
    const bool padded = p.negl_pad != nullptr;  // the producer fetches -L*log2e; else the warpgroup loads L itself
    float negl_next = (!padded && par < total) ? load_negl(par) : FAWS_NEG_INF;
    for (int u = par; u < total; u += 2, ++mine) {
      float* lb;
      if (padded) {
        lb = lbuf + (u % CS_LSLOTS) * BM;
        if (!mbar_wait(&bars->l_full[u % CS_LSLOTS], (u / CS_LSLOTS) & 1, abort_flag)) { alive = false; break; }
      } else {
        // Two L buffers per warpgroup: the barrier below completes only when every thread of the
        // warpgroup has finished the previous tile, so the buffer of the tile before that is free.
        lb = lbuf + (wg * 2 + (mine & 1)) * 128;
        lb[row] = negl_next;
        mbar_arrive(&bars->l_ready[wg]);
        if (u + 2 < total) negl_next = load_negl(u + 2);
        if (!mbar_wait(&bars->l_ready[wg], mine & 1, abort_flag)) { alive = false; break; }
      }
      if (!mbar_wait(&bars->s_full[wg], mine & 1, abort_flag)) { alive = false; break; }
      tc_fence_after();
      if (no_keys) {
        tc_fence_before();
        mbar_arrive(&bars->s_free[wg]);
        continue;
      }
      const int g = u / ntq, qt = qt0 + (u - g * ntq);
      const int i0 = qt * BM;
      // half tiles of queries that do not contribute (their -L is -inf) are left out
      const int c_begin = i0 + CS_CHUNK <= i_lo ? CS_CHUNK : 0, c_end = i0 + CS_CHUNK >= p.m_end && c_begin == 0 ? CS_CHUNK : BM;
      // causal: query column x is visible to key j iff i0 + x + p_seq >= j
      const int xlo = p.causal ? (j - p.p_seq - i0) : 0;
      const bool full = !p.causal || (nk0 + BN - 1 - p.p_seq - i0 <= 0);
      float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
#pragma unroll 1
      for (int c0 = c_begin; c0 < c_end; c0 += CS_CHUNK) {
        uint32_t r[CS_CHUNK];
#pragma unroll
        for (int c = 0; c < CS_CHUNK; c += 32)
          tmem_ld32(t_buf + c0 + c, reinterpret_cast<uint32_t(&)[32]>(r[c]));
        tmem_wait_ld();
        if (c0 + CS_CHUNK == c_end) {  // the buffer can take the next S^T of this warpgroup
          tc_fence_before();
          mbar_arrive(&bars->s_free[wg]);
        }
        const float* lh = lb + c0;
        if (full) {
          const uint64_t scale2 = pack_f32x2(scale_log2, scale_log2);
          uint64_t ap0 = pack_f32x2(a0, a1), ap1 = pack_f32x2(a2, a3);
#pragma unroll
          for (int x = 0; x < CS_CHUNK; x += 4) {
            const float4 nl = *reinterpret_cast<const float4*>(lh + x);
            float t0, t1, t2, t3;
            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(r[x]), __uint_as_float(r[x + 1])), scale2,
                                   pack_f32x2(nl.x, nl.y)), t0, t1);
            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(r[x + 2]), __uint_as_float(r[x + 3])), scale2,
                                   pack_f32x2(nl.z, nl.w)), t2, t3);
            ap0 = add_f32x2(ap0, pack_f32x2(fast_exp2(t0), fast_exp2(t1)));
            ap1 = add_f32x2(ap1, pack_f32x2(fast_exp2(t2), fast_exp2(t3)));
          }
          unpack_f32x2(ap0, a0, a1);
          unpack_f32x2(ap1, a2, a3);
        } else {
          const int xh = xlo - c0;
          // query columns below the smallest bound in the warp are hidden from all of its keys: no exp2 there
          const int xh_warp = __reduce_min_sync(0xffffffffu, xh);
#pragma unroll
          for (int x = 0; x < CS_CHUNK; x += 4) {
            if (x + 3 < xh_warp) continue;
            const float4 nl = *reinterpret_cast<const float4*>(lh + x);
            a0 += (x >= xh) ? fast_exp2(fmaf(__uint_as_float(r[x]), scale_log2, nl.x)) : 0.f;
            a1 += (x + 1 >= xh) ? fast_exp2(fmaf(__uint_as_float(r[x + 1]), scale_log2, nl.y)) : 0.f;
            a2 += (x + 2 >= xh) ? fast_exp2(fmaf(__uint_as_float(r[x + 2]), scale_log2, nl.z)) : 0.f;
            a3 += (x + 3 >= xh) ? fast_exp2(fmaf(__uint_as_float(r[x + 3]), scale_log2, nl.w)) : 0.f;
          }
        }
      }
      acc += (a0 + a1) + (a2 + a3);
    }
    if (!alive) acc = 0.f;
    if (par > 0) comb[kt * 128 + row] = acc;  // the odd query tiles' share of key tile kt
  }

  // ------------------------------------------------------------ common exit
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp >= 4 && warp < 4 + 4 * CS_KT) {  // the even-parity warpgroup of each key tile writes it
    const int row = (warp & 3) * 32 + lane;
    const int kt = (warp - 4) >> 2;
    const int j = n0 + kt * BN + row;
    if (j < p.n_end) {  // even query tiles first, then the odd ones
      p.out[((int64_t)b * n_heads_out + ho) * p.n_end + j] = acc + comb[kt * 128 + row];
    }
  }
  if (*abort_flag) {
    if (threadIdx.x == 0 && status != nullptr) atomicOr(status, 1);
    for (int w = 0; w < 50; ++w) __nanosleep(20000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------- host side
// Per-device status word the kernels raise when a bounded wait gives up.
__device__ int g_tc_status = 0;

}  // namespace

int* tc_status_word() {
  static int* words[kMaxDevices] = {nullptr};
  static std::mutex mu;
  const int dev = current_device();
  if (dev < 0) return nullptr;
  std::lock_guard<std::mutex> lock(mu);
  if (words[dev] == nullptr) {
    void* ptr = nullptr;
    if (cudaGetSymbolAddress(&ptr, g_tc_status) == cudaSuccess) words[dev] = static_cast<int*>(ptr);
  }
  return words[dev];
}

namespace {

// FAWS_SPLIT_KV=0/1 in the environment overrides the choice (tests, ablations).
template <int D, int HOOK>
bool use_split_kv(const FwdParams& p) {
  static const int forced = [] {
    const char* e = std::getenv("FAWS_SPLIT_KV");
    return e == nullptr ? -1 : (e[0] == '1' ? 1 : 0);
  }();
  if (forced >= 0) return forced == 1;
  const RowChoice c{(long long)p.B * p.Hq, p.m_begin, p.m_end, p.N, p.p_seq, p.causal, sm_count()};
  if (c.blocks(256) * c.heads >= 2LL * c.sms) return false;
  constexpr bool kStores = HOOK == kHookScores || HOOK == kHookScores16 || HOOK == kHookScoresAny;
  if (kStores || p.n_splits > 1 || p.pack_m > 0) return true;  // (the expected times know none of these)
  return !prefer_256_rows(c, D == 128, HOOK == kHookColPart ? kWithColSums : HOOK == kHookRowSum ? kWithRowSums : kPlainOut);
}

template <typename T, int D, int HOOK>
cudaError_t launch_fwd_h(const TcMaps& maps, const FwdParams& p, cudaStream_t s) {
  // Score-materialising causal launches with more CTAs than SMs are bound by their stores, not by the chain of key
  // tiles: measured, the 256-row CTAs (half as many set-ups) are faster there (fp16 D128 H32, 256 and 128 rows:
  // S1024 36.8 and 39.9 us, S768 27.0 and 26.5, S640 19.2 and 19.1).  When the 128-row CTAs all run at once the chain
  // is what counts again (D128 H16 S768 22.4 and 15.8 us, H8 S640 16.0 and 12.7; D64 H8 S512 15.9 and 10.6; H37 S512,
  // 148 CTAs, 19.1 and 15.8), but for three key tiles, which two warpgroups share badly, when nearly every SM has one
  // (D128 S384 H40 13.3 and 12.0, H44 13.2 and 13.2, H49 13.2 and 14.1).
  if constexpr (HOOK != kHookScores16 && HOOK != kHookScoresAny) {
    // Dropout: 256-row CTAs only.  Where the kernel draws the mask, that bounds it and not the chain of key tiles.  Where it reads
    // the mask there is no instance of 128-row CTAs, which would suit fewer of them than SMs (fp16 causal, mask kernel and
    // forward pass, 256 and 128 rows: B1 H16 S1000 D64 39.6 and 30.8 us, H8 S1900 D128 63.5 and 48.9; B2 H20 S1000 D64 60.1 and
    // 61.5, B4 H16 S300 25.0 and 26.1).
    if constexpr (HOOK == kHookNone) {
      if (p.drop_mask != nullptr)
        return p.mask_drawn ? launch_fwd_s<T, D, HOOK, false, kReadMask>(maps, p, s)
                            : launch_fwd_s<T, D, HOOK, false, kKeepMask>(maps, p, s);
    }
    if (p.drop.p > 0.f) return launch_fwd_s<T, D, HOOK, false, kDrawMask>(maps, p, s);
  }
  const long long ctas128 = (long long)((p.m_end - p.m_begin + 127) / 128) * p.Hq * p.B;
  // fp32 scores in odd rows: the line lies at 1.7 CTAs of 128 rows per SM (D128, 256 and 128 rows: H20 S1021, 160 of them,
  // 49.7 and 32.3 us; H16 S1531, 192, 70.3 and 50.6; H20 S1531, 240, 69.0 and 63.3; H32 S1021, 256, 51.2 and 49.5; H28
  // S1531, 336, 78.2 and 86.8).
  const bool odd_f32 = HOOK == kHookScoresAny && p.scores_f32;
  const bool store_bound = (HOOK == kHookScores || HOOK == kHookScores16 || HOOK == kHookScoresAny) && p.causal &&
                           (odd_f32 ? 3 * ctas128 > 5LL * sm_count()
                                    : ctas128 > ((p.N + BN - 1) / BN == 3 ? sm_count() * 7 / 8 : sm_count()));
  // Without a mask 256-row CTAs take some 1.65 times as long as 128-row ones, so whole waves decide (D128 full, 256 and 128
  // rows: H24 S1531, 144 and 288 CTAs, 76.1 and 97.6 us; H28, 168 and 336, 147 and 129).  Over 156 odd shapes of 1 to 2.9 CTAs of
  // 128 rows per SM, D 32 to 128, what both rules take is 0.5 % behind the better of the two in the mean; the worst: one row
  // beyond a 256-row CTA (causal H84 S257 27.2 us, 22.3 with 128 rows), causal just above the line (H32 S1021 D64 49.1 and 45.7),
  // full just above one wave (H26 S641 D32 34.3 and 32.3, H15 S1163 D128 58.7 and 56.3).
  const long long ctas256 = (long long)((p.m_end - p.m_begin + 255) / 256) * p.Hq * p.B;
  const bool fewer_waves = odd_f32 && !p.causal &&
                           5 * ((ctas256 + sm_count() - 1) / sm_count()) <= 3 * ((ctas128 + sm_count() - 1) / sm_count());
  static const bool forced = std::getenv("FAWS_SPLIT_KV") != nullptr;
  const bool split = use_split_kv<D, HOOK>(p) && (forced || !(store_bound || fewer_waves));
  if constexpr (HOOK == kHookNone) {
    if (p.pack_m > 0 || p.n_splits > 1)
      return split ? launch_fwd_s<T, D, HOOK, true, kNoDrop, true>(maps, p, s)
                   : launch_fwd_s<T, D, HOOK, false, kNoDrop, true>(maps, p, s);
  }
  return split ? launch_fwd_s<T, D, HOOK, true>(maps, p, s) : launch_fwd_s<T, D, HOOK, false>(maps, p, s);
}

template <typename T, int D>
cudaError_t launch_fwd_t(const TcMaps& maps, const FwdParams& p, cudaStream_t s) {
  if (p.scores != nullptr && !tma_score_rows(p.scores, p.N, p.scores_f32 ? 4 : 2))
    return launch_fwd_h<T, D, kHookScoresAny>(maps, p, s);
  if (p.scores != nullptr)
    return p.scores_f32 ? launch_fwd_h<T, D, kHookScores>(maps, p, s) : launch_fwd_h<T, D, kHookScores16>(maps, p, s);
  if (p.row_sum != nullptr) return launch_fwd_h<T, D, kHookRowSum>(maps, p, s);
  if (p.col_partial != nullptr) return launch_fwd_h<T, D, kHookColPart>(maps, p, s);
  return launch_fwd_h<T, D, kHookNone>(maps, p, s);
}

}  // namespace

bool tc_fwd_supported(const FwdParams& p, int dtype) {
  (void)dtype;
  if (!tc_head_dim(p.D)) return false;
  if (p.s_scratch != nullptr) return false;  // the score buffer of the cross-token operator: CUDA-core kernels only
  if (p.drop.p > 0.f && p.scores != nullptr && !p.scores_f32)
    return false;  // no dropout variant of the 16-bit-score hook: CUDA-core kernels
  if (!(p.sm_scale > 0.f)) return false;  // the row max is taken on unscaled scores
  if (!device_is_sm100() || get_encode() == nullptr) return false;
  if (p.m_begin % BM != 0 || p.m_end <= p.m_begin) return false;
  if (!ok16(p.q, p.q_sb, p.q_sh, p.q_ss) || !ok16(p.k, p.k_sb, p.k_sh, p.k_ss) ||
      !ok16(p.v, p.v_sb, p.v_sh, p.v_ss) || !ok16(p.o, p.o_sb, p.o_sh, p.o_ss))
    return false;
  if (p.scores != nullptr && !tma_score_rows(p.scores, p.N, p.scores_f32 ? 4 : 2)) {
    if (p.drop.p > 0.f) return false;  // the plain-store hook has no dropout variant
    if (reinterpret_cast<uintptr_t>(p.scores) % (p.scores_f32 ? 4 : 2) != 0) return false;
  }
  return true;
}

cudaError_t launch_tc_fwd(const FwdParams& p, int dtype, cudaStream_t s) {
  if (p.window > 0) return launch_tc_fwd_window(p, dtype, s);
  TcMaps maps;
  if (!make_fwd_maps(&maps, p)) return cudaErrorInvalidValue;
  if (dtype == FAWS_FP16)
    return p.D == 128 ? launch_fwd_t<__half, 128>(maps, p, s) : launch_fwd_t<__half, 64>(maps, p, s);
  return p.D == 128 ? launch_fwd_t<__nv_bfloat16, 128>(maps, p, s) : launch_fwd_t<__nv_bfloat16, 64>(maps, p, s);
}

namespace {
// Exercises the give-up path of mbar_wait: one thread waits (bounded, about a millisecond) on an
// mbarrier nobody arrives at, the wait runs out, the CTA raises the status word and returns.
__global__ void wait_give_up_kernel(int* __restrict__ status, long long limit_cycles) {
  __shared__ uint64_t bar;
  __shared__ int abort_flag;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (threadIdx.x == 0) mbar_wait(&bar, 0, &abort_flag, limit_cycles);
  __syncthreads();
  if (abort_flag != 0 && threadIdx.x == 0 && status != nullptr) atomicOr(status, 1);
}
}  // namespace

cudaError_t launch_wait_give_up(cudaStream_t s) {
  int* status_word = tc_status_word();
  if (status_word == nullptr) return cudaErrorInvalidDevice;
  wait_give_up_kernel<<<1, 32, 0, s>>>(status_word, 2000000ll);
  count_launch();
  return cudaGetLastError();
}

int tc_read_status(int reset) {
  int* word = tc_status_word();
  if (word == nullptr) return -1;
  int v = 0;
  if (cudaMemcpy(&v, word, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return -1;
  if (reset && v != 0) cudaMemset(word, 0, sizeof(int));
  return v;
}

// Whether the kernel should walk the G heads of a kv head inside one CTA (output already group
// summed) or run one CTA per query head followed by a group-sum kernel.  The latter gives G times
// more CTAs, which matters for causal problems where the key tiles' work is very uneven.
bool tc_colsoftmax_group_in_kernel(const ColSoftmaxParams& p) {
  if (p.G == 1) return true;
  const int sms = sm_count();
  const long long ctas = (long long)((p.n_end + CS_KT * BN - 1) / (CS_KT * BN)) * p.Hk * p.B;
  return !(p.causal && ctas < 8LL * sms) && ctas >= 2LL * sms;
}

bool tc_colsoftmax_supported(const ColSoftmaxParams& p, int dtype) {
  (void)dtype;
  if (!tc_head_dim(p.D)) return false;
  if (p.s_scratch != nullptr) return false;  // the buffered pass reads stored scores, no MMA
  if (p.drop.p > 0.f) return false;
  if (p.m_begin % BM != 0 || !(p.sm_scale > 0.f)) return false;
  if (!device_is_sm100() || get_encode() == nullptr) return false;
  if (!ok16(p.q, p.q_sb, p.q_sh, p.q_ss) || !ok16(p.k, p.k_sb, p.k_sh, p.k_ss)) return false;
  return p.n_end > 0;
}

namespace {
// -L_i*log2e into the tile-padded array the key-major kernel copies from; -inf for rows that do not
// contribute (outside [i_lo, m_end), padding, or without a visible key).
__global__ void negl_prep_kernel(const float* L, float* out, int M, int m_pad, int i_lo,
                                 int m_end, long long total) {
  griddep_wait();  // L comes from the forward pass before this launch
  griddep_launch_dependents();
  const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (idx >= total) return;
  const long long bh = idx / m_pad;
  const int i = (int)(idx - bh * m_pad);
  float v = FAWS_NEG_INF;
  if (i >= i_lo && i < m_end) {
    const float Li = L[bh * M + i];
    if (Li != FAWS_NEG_INF) v = -Li * kLog2e;
  }
  out[idx] = v;
}

cudaError_t launch_negl_prep(const ColSoftmaxParams& p, cudaStream_t s) {
  const long long total = (long long)p.B * p.Hq * p.m_pad;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((total + 255) / 256), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.after_forward ? 1 : 0;
  const float* L = p.L;
  float* out = p.negl_pad;
  const int i_lo = p.i_begin > p.m_begin ? p.i_begin : p.m_begin;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, negl_prep_kernel, L, out, p.M, p.m_pad, i_lo, p.m_end, total);
  count_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int D>
cudaError_t launch_cs_t(const CsMaps& maps, const ColSoftmaxParams& call, int heads_per_cta, cudaStream_t s) {
  ColSoftmaxParams p = call;
  using L = CsSmem<D>;
  static PerDeviceOnce attr_once;
  if (cudaError_t e = set_max_smem_once(attr_once, tc_colsoftmax_kernel<T, D>, L::alloc); e != cudaSuccess) return e;
  const int nkt = (p.n_end + CS_KT * BN - 1) / (CS_KT * BN);  // CTAs along the keys: CS_KT key tiles each
  // A head's last CTA of one key tile at most, which takes half as long: last (fp16 B16 H8 S785 D32, 17 of 256 keys, with the
  // forward pass 104.8 -> 103.4 us, B4 H32 S300 D128 39.9 -> 36.4); as long as the queries stay in L2, so that the CTAs of a
  // head need not run together.  The order is that of a causal launch, and a causal launch whose queries all see every key
  // is a full one: the kernel need not tell them apart (a field for the order cost it registers, and causal launches 0.5 %).
  const int last = p.n_end - (nkt - 1) * CS_KT * BN;
  if (!p.causal && last <= BN && nkt > 1 && nkt <= 65535 && 2LL * p.B * p.Hq * p.m_end * p.D <= (48LL << 20)) {
    p.causal = 1;
    p.p_seq = nkt * CS_KT * BN;
  }
  dim3 grid = p.causal ? dim3(p.Hq / heads_per_cta, p.B, nkt) : dim3(nkt, p.Hq / heads_per_cta, p.B);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(CS_THREADS, 1, 1);
  cfg.dynamicSmemBytes = L::alloc;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.after_forward ? 1 : 0;  // q and k must not come from the previous kernel
  int* status_word = tc_status_word();
  const cudaError_t e = cudaLaunchKernelEx(&cfg, tc_colsoftmax_kernel<T, D>, maps, p, heads_per_cta, status_word);
  count_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}
}  // namespace

// group_sum != 0: one CTA walks the G query heads of a kv head and p.out is (B,Hk,n_end);
// otherwise one CTA per query head and p.out is (B,Hq,n_end).
cudaError_t launch_tc_colsoftmax(const ColSoftmaxParams& call, int dtype, int group_sum, cudaStream_t s) {
  ColSoftmaxParams p = call;
  CsMaps maps;
  if (!make_map_bhsd(&maps.q, p.q, p.D, p.m_end, p.Hq, p.B, p.q_ss, p.q_sh, p.q_sb, 128) ||
      !make_map_bhsd(&maps.k, p.k, p.D, p.N, p.Hk, p.B, p.k_ss, p.k_sh, p.k_sb, 128))
    return cudaErrorInvalidValue;
  const int hpc = group_sum ? p.G : 1;
  // A CTA of few query tiles loads L itself: the launch that lays it out for bulk copies takes longer than it saves, and
  // stands between this kernel's set-up and the forward pass.  fp16 H32 D128 causal, S256 split 192, one tile: 15.7 us with
  // it, 12.5 without; four tiles 8 % faster without, eight 2.6 %, ten the same, sixteen 2 % slower.
  const int i_lo = p.i_begin > p.m_begin ? p.i_begin : p.m_begin;
  if (hpc * ((p.m_end + BM - 1) / BM - i_lo / BM) <= 8) p.negl_pad = nullptr;
  if (p.negl_pad != nullptr) {
    if (cudaError_t e = launch_negl_prep(p, s); e != cudaSuccess) return e;
  }
  if (dtype == FAWS_FP16)
    return p.D == 128 ? launch_cs_t<__half, 128>(maps, p, hpc, s) : launch_cs_t<__half, 64>(maps, p, hpc, s);
  return p.D == 128 ? launch_cs_t<__nv_bfloat16, 128>(maps, p, hpc, s)
                    : launch_cs_t<__nv_bfloat16, 64>(maps, p, hpc, s);
}

}  // namespace faws
