// Attention of many query rows over a paged 8-bit cache (csrc/kv8.cuh), on the
// fifth-generation tensor cores. 16-bit operands, head dimensions up to 128.
//
// A CTA takes 256 query rows (tokens x heads of a kv head's group) of one
// sequence and kv head, as two tiles of 128, and goes over the tokens in
// blocks of 64:
//   S_i = Q_i K^T (tcgen05, fp32 in TMEM)  ->  softmax warps of tile i
//   P_i = 2^(S f - m) as fp16, in TMEM  ->  O_i += P_i V (A from TMEM)
// S is free for the next block's scores as soon as its warps have it in
// registers, so that they never wait for the way through the tensor cores and
// back. An MMA with both operands in shared memory is bound by reading them
// (97 clocks for 128 x 64 x 16 against 32 of arithmetic): the first 64 elements
// of the rows of Q lie in TMEM, which is then full.
// Keys and values come as raw codes by bulk copies and are decoded once for
// all 256 rows into swizzled fp16 operands (exact). Rows of q are scaled to
// 2^13..2^14 by a power of two (exact for 16-bit types down to 2^-27 of the
// row's largest value). Page scales: f = sk x the row's power x scale goes into
// the exponent, and so do values' scales: a weight is 2^(S f + log2 sv - m), its
// sum is taken back by 2^-log2 sv, and what a row does not see, or gives no
// weight to, takes no bits from what it sees. The maximum m (of S f + log2 sv) is
// taken 2^3 above the block's when it is set, and O is rescaled in TMEM only when
// it moves: where a weight would pass 2^8, or, in blocks with hidden tokens or odd
// scales, 1. Weights (times 2^7) stay below 2^15, fp16 rounds them by 2^-11,
// sums are fp32.
//
// What bounds it: for 64 tokens and 256 rows the MMAs take about 1550 clocks
// (the half of Q in shared memory most of it), the exponentials 1024; the way
// from scores through a tile's softmax to P and back is longer than both, so
// that it takes 2400. bf16, 2 x 1000 over 8000, 32 heads: 297 us, 0.60 PFLOP/s of
// the products it needs, with 1.73 CTAs an SM in two rounds. Blocks of 128
// tokens with one S, both operands in shared memory, took 365.
// Roles: warps 0-3 and 4-7 softmax of tiles 0 and 1 (a thread a row), 8-11
// decode, 12 copies, 13 and 14 issue the MMAs of tiles 0 and 1.
#pragma once
#include "kv8_attn.cuh"
#include "q4_gemm.cuh"

namespace tt {
namespace kv8 {

// Sums of values stay in the tensor cores, which cut off up to 2^-23 of them at
// every 16 tokens, to one side. Where a table can hold so many that a result
// would show it, a tile's rows put O aside every kLongRun blocks, in a place of
// the workspace that the CTA takes when it starts, and the next block starts anew.
constexpr int kPreThreads = 15 * 32;
constexpr int kPreKeys = 64;         // tokens of a block
constexpr int kPreBufs = 4;          // decoded blocks of K and of V
constexpr int kScaleSlots = 8;       // the copies are at most six blocks ahead of the softmax
constexpr float kPreUp = 128.f, kPreUpLog = 7.f;  // a weight of 1 in P
constexpr float kPreRoom = 3.f;      // m above the largest score when it is set, and
constexpr float kPreRise = 8.f;      // a score above m that it bears; both as powers of two

template <int DP>
struct PreShape {
  static constexpr int kQ = 128 * (DP - 64) * 2;      // bytes of a tile of Q behind element 64
  static constexpr int kKV = kPreKeys * DP * 2;       // of K or V as fp16
  static constexpr int kRaw = kPreKeys * DP;          // and as codes
  static constexpr int kSmem = 2 * kQ + 2 * kPreBufs * kKV + 4 * kRaw + 1024;
  // first columns of tile 0; tile 1 is as many behind as one takes
  static constexpr int kS = 0, kP = 128, kQt = 192, kO = 256;
  static_assert(kSmem + 1280 + 512 <= 227 * 1024, "shared memory of an SM");
};

// D[tmem] (+)= A[tmem] B[smem]^T, fp16 operands.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tmov.b64 y, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(q4::kDescHigh)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8u(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// kFull: the head dimension is DP. kLong: O is put aside (its code costs the
// others 3 to 13% of their time, by registers; 1000 rows over 60000 tokens in
// fp16 1372 us, without it 1290).
template <typename T, int DP, bool kFull, bool kLong>
__global__ void __launch_bounds__(kPreThreads, 1) prefill_kernel(const Attend p) {
  using S = PreShape<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sm_q = smem;
  uint8_t* sm_k = sm_q + 2 * S::kQ;
  uint8_t* sm_v = sm_k + kPreBufs * S::kKV;
  uint8_t* sm_raw = sm_v + kPreBufs * S::kKV;
  constexpr int kUnits = kPreKeys / 16;
  // of block j: [..][j % 2], in its phase j / 2 % 2, or with kPreBufs for 2
  __shared__ uint64_t raw_full[2][2], raw_empty[2][2], k_full[kPreBufs], k_empty[kPreBufs], v_full[kPreBufs],
      v_empty[kPreBufs], q_ready, last;
  // of tile i, in the phase j % 2 of block j
  __shared__ uint64_t s_full[2], s_free[2], p_full[2], pv_done[2];
  // keys' scales, and values' (Level)
  __shared__ float sc_k[kScaleSlots][kUnits], sc_odd[kScaleSlots][kUnits], sc_log[kScaleSlots][kUnits],
      sc_inv[kScaleSlots][kUnits];
  __shared__ uint32_t tmem_slot;
  __shared__ int dead, top_lim, before, place;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int dim = kFull ? DP : p.dim, group = p.heads_q / p.heads;
  const int b = blockIdx.z, h = blockIdx.y;
  const int tile = gridDim.x - 1 - blockIdx.x;  // the longest first
  const int tiles = p.rows - tile * 256 > 128 ? 2 : 1;
  const int length = (int)clamp_length(p, b, threadIdx.x == 0 && h == 0 && blockIdx.x == 0);
  const int count = clamp_count(p, b, threadIdx.x == 0 && h == 0 && blockIdx.x == 0);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      for (int k = 0; k < 2; ++k) {
        mbar_init(&raw_full[i][k], 1);
        mbar_init(&raw_empty[i][k], 4);
      }
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < kPreBufs; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&k_empty[i], tiles);
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], tiles);
    }
    mbar_init(&q_ready, 256);
    mbar_init(&last, tiles);
    fence_mbar_init();
    dead = 0;
    top_lim = 0;
    before = 0;
    place = -1;
  }
  if (warp == 13) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  __syncthreads();
  // rows of this thread (softmax warps), and what they see
  int lim = 0, row = -1;
  const T* from = nullptr;
  if (warp < 8) {
    const int r = tile * 256 + threadIdx.x;
    if (r < p.rows) {
      row = r;
      const int tok = r / group, head = h * group + r % group;
      if (tok < count) {
        lim = max(p.causal ? length - count + tok + 1 : length, 0);
        from = static_cast<const T*>(p.q) + b * p.q_b + tok * p.q_s + head * p.q_h;
      }
    }
    const int most = __reduce_max_sync(0xffffffffu, lim);
    if (lane == 0) atomicMax(&top_lim, most);
  }
  __syncthreads();
  const int blocks = (top_lim + kPreKeys - 1) / kPreKeys;
  if (kLong && top_lim > p.most && threadIdx.x == 0) {
    // No more CTAs than places run at a time (were there none free, O would stay);
    // the first to ask for is this SM's.
    uint32_t sm;
    asm volatile("mov.u32 %0, %%smid;" : "=r"(sm));
    int at = (int)(sm % (uint32_t)p.sms), left = p.sms;
    while (left > 0 && atomicCAS(p.places + at, 0, 1) != 0) {
      at = at + 1 == p.sms ? 0 : at + 1;
      --left;
    }
    if (left > 0) place = at;
    __threadfence();
  }
  if (dim < DP) {  // columns of K and Q behind the head dimension are zeros, for good
    for (int i = threadIdx.x; i < (2 * S::kQ + kPreBufs * S::kKV) / 16; i += kPreThreads)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  int* err = &dead;

  if (warp == 12) {
    // ---- copies: a lane a unit of 16 tokens
    for (int j = 0; j < blocks; ++j) {
      const int tok = j * kPreKeys + 16 * lane, buf = j & 1, phase = (j >> 1) & 1;
      int page = -1;
      if (lane < kUnits && tok < length) page = p.table[b * p.table_b + (tok >> p.page_log)];
      const bool gone = lane < kUnits && tok < length && (page < 0 || page >= p.pages);
      if (gone) {
        raise(p.status, kBadPage);
        page = -1;
      }
      const long long head = (long long)max(page, 0) * p.heads + h;
      if (lane < kUnits) {
        sc_k[j % kScaleSlots][lane] = page >= 0 ? p.ks[head] : gone ? kGone : 0.f;
        const Level sv = level_of<false>(page >= 0 ? p.vs[head] : 0.f, kPreUp);
        sc_odd[j % kScaleSlots][lane] = sv.odd;
        sc_log[j % kScaleSlots][lane] = sv.lg;
        sc_inv[j % kScaleSlots][lane] = sv.back;
      }
      __syncwarp();  // before lane 0's arrival below, which the softmax warps wait behind
      const unsigned has = __ballot_sync(0xffffffffu, page >= 0);
      const long long at = (head * p.page + (tok & (p.page - 1))) * dim;
      bool ok = true;
      for (int v = 0; v < 2 && ok; ++v) {
        ok = __all_sync(0xffffffffu, mbar_wait(&raw_empty[v][buf], phase ^ 1, err, kTimeout));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&raw_full[v][buf], __popc(has) * 16 * dim);
        __syncwarp();
        if (page >= 0)
          bulk_load(smem_u32(sm_raw + (2 * v + buf) * S::kRaw + lane * 16 * dim), (v ? p.vc : p.kc) + at, 16 * dim,
                    smem_u32(&raw_full[v][buf]));
      }
      if (!ok) break;
    }
    // what is in flight arrives, or the wait for it is over
    if (lane == 0 && dead != 0)
      for (int j = max(blocks - 2, 0); j < blocks; ++j)
        for (int v = 0; v < 2; ++v) mbar_wait_drain(&raw_full[v][j & 1], (j >> 1) & 1);
    __syncwarp();
  } else if (warp >= 13) {
    // ---- MMAs, a warp a tile: it goes together, one lane issues
    const int i = warp - 13;
    // a copy of an earlier call never arrived, and nobody has looked at that yet
    if (i == 0 && lane == 0) *(volatile int*)&before = *(volatile int*)p.status & kTimeout;
    if (blocks > 0 && i < tiles) {
      constexpr uint32_t id_s = q4::idesc_f16(128, kPreKeys, 0), id_o = q4::idesc_f16(128, DP, 0);
      const uint32_t q = q4::desc_low(smem_u32(sm_q + i * S::kQ)), k0 = q4::desc_low(smem_u32(sm_k)),
                     v0 = q4::desc_low(smem_u32(sm_v)), d0 = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t ds = d0 + S::kS + i * kPreKeys, dq = d0 + S::kQt + i * 32, dp = d0 + S::kP + i * 32,
                     o = d0 + S::kO + i * DP;
      auto scores = [&](int buf) {  // S of the block in `buf`
        const uint32_t k = k0 + buf * (S::kKV >> 4);
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_f16_ts(ds, dq + s * 8, k + s * 2, id_s, s != 0);
#pragma unroll
          for (int s = 4; s < DP / 16; ++s)
            q4::mma_f16(ds, q + (s - 4) * 2, k + (kPreKeys * 128 >> 4) + (s - 4) * 2, id_s, 1);
          mma_commit(&s_full[i]);
          mma_commit(&k_empty[buf]);
        }
        __syncwarp();
      };
      auto values = [&](int buf, bool first) {  // O += P V
        const uint32_t v = v0 + buf * (S::kKV >> 4);
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < kPreKeys / 16; ++s) mma_f16_ts(o, dp + s * 8, v + s * 2, id_o, !first || s != 0);
          mma_commit(&pv_done[i]);
          mma_commit(&v_empty[buf]);
        }
        __syncwarp();
      };
      auto ready = [&](uint64_t* bar, int phase) {
        const bool here = __all_sync(0xffffffffu, mbar_wait(bar, phase, err, kTimeout));
        tc_fence_after();
        return here;
      };
      bool ok = ready(&q_ready, 0) && ready(&k_full[0], 0);
      if (ok) scores(0);
      for (int j = 0; j < blocks && ok; ++j) {
        if (j + 1 < blocks) {  // the next block's scores, before the softmax of this one ends
          const int n = (j + 1) % kPreBufs, phase = (j + 1) / kPreBufs & 1;
          ok = ready(&k_full[n], phase) && ready(&s_free[i], j & 1);
          if (!ok) break;
          scores(n);
        }
        ok = ready(&v_full[j % kPreBufs], j / kPreBufs & 1) && ready(&p_full[i], j & 1);
        if (ok) values(j % kPreBufs, j == 0 || (kLong && place >= 0 && j % kLongRun == 0));
      }
      // nothing may be in flight when the CTA gives its TMEM back
      if (elect_one()) {
        mma_commit(&last);
        mbar_wait_drain(&last, 0);
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    // ---- decoding
    const int id = threadIdx.x - 256;
    bool ok = true;
    for (int j = 0; j < blocks && ok; ++j) {
      const int from_buf = j & 1, buf = j % kPreBufs;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        ok = mbar_wait(&raw_full[v][from_buf], (j >> 1) & 1, err, kTimeout) &&
             mbar_wait(v ? &v_empty[buf] : &k_empty[buf], (j / kPreBufs & 1) ^ 1, err, kTimeout);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t raw = smem_u32(sm_raw + (2 * v + from_buf) * S::kRaw);
        const uint32_t to = smem_u32((v ? sm_v : sm_k) + buf * S::kKV);
        const int wide = kFull ? DP : dim;  // kFull: all divisions below are shifts
        const int per = wide / 16, all = kPreKeys * per;  // pieces of 16 codes
#pragma unroll 8
        for (int i = id; i < all; i += 128) {
          const uint4 q = lds128(raw + i * 16);
          uint32_t w[8];
          decode4(q.x, w[0], w[1]);
          decode4(q.y, w[2], w[3]);
          decode4(q.z, w[4], w[5]);
          decode4(q.w, w[6], w[7]);
          if (v) {
            // unit u, d: sixteen tokens of it, in line d of the operand
            const uint32_t u = i / wide, r = i % wide;
            const uint32_t line = to + r * 128, c = u * 2;
            sts128(line + ((c ^ (r & 7)) << 4), w[0], w[1], w[2], w[3]);
            sts128(line + (((c + 1) ^ (r & 7)) << 4), w[4], w[5], w[6], w[7]);
          } else {
            // a token, sixteen d of it; from 64 on the second half first:
            // eight lanes then meet all banks
            const uint32_t r = i / per, x = i % per;
            const uint32_t line = to + x / 4 * (kPreKeys * 128) + r * 128, c = x % 4 * 2, swap = x / 4 & 1;
            sts128(line + (((c + swap) ^ (r & 7)) << 4), swap ? w[4] : w[0], swap ? w[5] : w[1], swap ? w[6] : w[2],
                   swap ? w[7] : w[3]);
            sts128(line + (((c + 1 - swap) ^ (r & 7)) << 4), swap ? w[0] : w[4], swap ? w[1] : w[5],
                   swap ? w[2] : w[6], swap ? w[3] : w[7]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&raw_empty[v][from_buf]);
          mbar_arrive(v ? &v_full[buf] : &k_full[buf]);
        }
      }
    }
  } else {
    // ---- softmax: a thread a row
    const int i = warp >> 2;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float qs;
    {  // this row of Q
      float top = 0.f;
      uint4 raw[DP / 8];  // all loads go out together
#pragma unroll
      for (int c = 0; c < DP / 8; ++c)
        raw[c] = from != nullptr && 8 * c < dim ? __ldg(reinterpret_cast<const uint4*>(from) + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < DP / 8; ++c) {
        const T* x = reinterpret_cast<const T*>(&raw[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(q4::to_f(x[e])));
      }
      int ex = (int)((__float_as_uint(top) >> 23) & 255);
      ex = ex < 14 ? 14 : ex;
      const float up = __uint_as_float((uint32_t)(267 - ex) << 23) * (p.scale < 0.f ? -1.f : 1.f);
      qs = __uint_as_float((uint32_t)(ex - 13) << 23) * fabsf(p.scale);
      const uint32_t r = threadIdx.x & 127;
#pragma unroll
      for (int d = 0; d < DP; d += 16) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const T* x = reinterpret_cast<const T*>(&raw[d / 8]) + 2 * e;
          w[e] = q4::pack_f16(q4::to_f(x[0]) * up, q4::to_f(x[1]) * up);
        }
        __syncwarp();
        if (d < 64) {
          tmem_st8u(lane_base + S::kQt + i * 32 + d / 2, w);
        } else {
          const uint32_t line = smem_u32(sm_q + i * S::kQ) + r * 128, c = d % 64 / 8;
          sts128(line + ((c ^ (r & 7)) << 4), w[0], w[1], w[2], w[3]);
          sts128(line + (((c + 1) ^ (r & 7)) << 4), w[4], w[5], w[6], w[7]);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      fence_proxy_async_smem();
      mbar_arrive(&q_ready);
    }
    const uint32_t to = lane_base + S::kO + i * DP, ts = lane_base + S::kS + i * kPreKeys, tp = lane_base + S::kP + i * 32;
    // the least that a row of this warp which sees anything sees
    int least = lim > 0 ? lim : 0x7fffffff;
    least = __reduce_min_sync(0xffffffffu, least);
    // a row that sees nothing stays out of the maxima's way
    float m = lim > 0 ? -INFINITY : 0.f, l = 0.f;
    bool ok = true;
    // O put aside, relative to the maximum at that time
    float m_aside = -INFINITY;
    float* aside = !kLong || place < 0 ? nullptr : p.aside + (long long)place * 256 * dim + threadIdx.x;
    auto put_aside = [&]() {
      const float z = m == -INFINITY ? 0.f : m, keep = exp2_approx(m_aside - z);
#pragma unroll 1
      for (int c = 0; c < dim; c += 16) {
        float o[16];
        tmem_ld16(to + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float* at = aside + (c + e) * 256;
          *at = m_aside == -INFINITY ? o[e] : fmaf(*at, keep, o[e]);
        }
      }
      m_aside = z;
    };
    // rows whose maximum rises, to a new one above n: l and O follow
    auto lift = [&](bool rise, float n, bool first) {
      const float now = rise ? n + kPreRoom : m;
      const float z = now == -INFINITY ? 0.f : now;
      const float a = m == -INFINITY ? 0.f : exp2_approx(m - z);
      l *= a;
      m = now;
      if (first) return;
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        float o[2][16];
        tmem_ld16(to + c, o[0]);
        tmem_ld16(to + c + 16, o[1]);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e / 16][e % 16] *= rise ? a : 1.f;
        tmem_st16(to + c, o[0]);
        tmem_st16(to + c + 16, o[1]);
      }
      tmem_st_wait();
    };
    if (i < tiles) {
      for (int j = 0; j < blocks; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[i], j & 1, err, kTimeout));
        if (!ok) break;
        tc_fence_after();
        if (kLong && aside != nullptr && j > 0 && j % kLongRun == 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[i], (j - 1) & 1, err, kTimeout));
          if (!ok) break;
          tc_fence_after();
          put_aside();
        }
        const float* fk = sc_k[j % kScaleSlots];
        // values' scales: their logarithms, inverses, and what is left of odd ones
        const float* fo = sc_odd[j % kScaleSlots];
        const float* fl = sc_log[j % kScaleSlots];
        const float* fi = sc_inv[j % kScaleSlots];
        const int tok0 = j * kPreKeys;
        const bool mask = tok0 + kPreKeys > least;
        uint32_t w[2][16];
        float n = -INFINITY;
        // Nothing hidden, and a maximum to go by.
        if (!mask && __all_sync(0xffffffffu, m != -INFINITY)) {  // the warp goes together
          bool plain = true;
          float sum = 0.f;
          float s[2][32];
          tmem_ld32(ts, s[0]);
          tmem_ld32(ts + 32, s[1]);
          tmem_ld_wait();
#pragma unroll
          for (int u = 0; u < kUnits; ++u) {
            const float* x = s[u / 2] + 16 * (u & 1);
            float t[4];
            plain = plain && fo[u] == 1.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = fmaxf(fmaxf(x[e], x[e + 4]), fmaxf(x[e + 8], x[e + 12]));
            n = fmaxf(n, fmaf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), qs * fk[u], fl[u]));
          }
          // units of odd scales, and those that are not there (their values' scale is 0), come below
          if (__all_sync(0xffffffffu, plain)) {
            tc_fence_before();
            if (lane == 0) mbar_arrive(&s_free[i]);
            __syncwarp();
            const bool rise = lim > 0 && n > m + kPreRise;
            if (__any_sync(0xffffffffu, rise)) {
              if (j > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[i], (j - 1) & 1, err, kTimeout));
                if (!ok) break;
                tc_fence_after();
              }
              lift(rise, n, j == 0);
            }
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
              float* x = s[u / 2] + 16 * (u & 1);
              const float f = qs * fk[u], y = fl[u] + (kPreUpLog - m);
              float q[4];
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e] = exp2_approx(fmaf(x[e], f, y));
#pragma unroll
              for (int e = 0; e < 4; ++e) q[e] = (x[e] + x[e + 4]) + (x[e + 8] + x[e + 12]);
              sum = fmaf((q[0] + q[1]) + (q[2] + q[3]), fi[u], sum);
#pragma unroll
              for (int e = 0; e < 8; ++e) w[u / 2][8 * (u & 1) + e] = q4::pack_f16(x[2 * e], x[2 * e + 1]);
            }
            l += sum;
            if (j > 0) {  // P of the block before has been read
              ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[i], (j - 1) & 1, err, kTimeout));
              if (!ok) break;
              tc_fence_after();
            }
            tmem_st16u(tp, w[0]);
            tmem_st16u(tp + 16, w[1]);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[i]);
            continue;
          }
        }
        // First blocks, hidden tokens, odd scales.
        n = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float s[32];
          tmem_ld32(ts + 32 * c, s);
          tmem_ld_wait();
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float sk = fk[2 * c + u];
            const int end = sk < 0.f ? 0 : lim;  // nothing is seen of a page that is not there
            float t = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (tok0 + 32 * c + 16 * u + e < end) t = fmaxf(t, s[16 * u + e]);
            // a hidden unit of scale 0 is not a number, and drops out
            n = fmaxf(n, fmaf(t, qs * (sk < 0.f ? 0.f : sk), fl[2 * c + u]));
          }
        }
        if (j > 0) {  // P of the block before has been read, and O is there to be rescaled
          ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[i], (j - 1) & 1, err, kTimeout));
          if (!ok) break;
          tc_fence_after();
        }
        const bool rise = n > m + kPreRise;  // from -inf: always, where anything is seen
        if (__any_sync(0xffffffffu, rise)) lift(rise, n, j == 0);
        const float z = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float s[32];
          tmem_ld32(ts + 32 * c, s);
          tmem_ld_wait();
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float* x = s + 16 * u;
            const float f = qs * fk[2 * c + u], y = fl[2 * c + u] + (kPreUpLog - z), odd = fo[2 * c + u];
            const int end = fk[2 * c + u] < 0.f ? 0 : lim;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const bool hidden = tok0 + 32 * c + 16 * u + e >= end;
              const float v = hidden ? 0.f : exp2_approx(fmaf(x[e], f, y));
              sum += v;
              x[e] = hidden ? 0.f : v * odd;
            }
            l = fmaf(sum, fi[2 * c + u], l);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[c][8 * u + e] = q4::pack_f16(x[2 * e], x[2 * e + 1]);
          }
          tmem_st16u(tp + 16 * c, w[c]);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s_free[i]);
          mbar_arrive(&p_full[i]);
        }
      }
      // `last` has one phase only. (pv_done could go on to the next phase, and
      // look unfinished, before a slow warp asks for the one before.)
      if (ok && blocks > 0) ok = __all_sync(0xffffffffu, mbar_wait(&last, 0, err, kTimeout));
      tc_fence_after();
    }
    const bool some = lim > 0 && blocks > 0;
    // then, or where a wait ran out here, the result is not a number
    const bool lost = !ok || *(volatile int*)&dead != 0 || *(volatile int*)&before != 0;
    const float inv = lost ? __int_as_float(0x7fffffff) : some && (l > 0.f || l != l) ? 1.f / (l * kPreUp) : 0.f;
    const float keep = exp2_approx(m_aside - (m == -INFINITY ? 0.f : m));
    for (int c = 0; c < dim; c += 16) {
      float o[16];
      if (blocks > 0 && i < tiles) {
        tmem_ld16(to + c, o);
        tmem_ld_wait();
        if (kLong && aside != nullptr) {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = fmaf(aside[(c + e) * 256], keep, o[e]);
        }
      }
      if (row >= 0) {
        T* at = static_cast<T*>(p.o) + row_offset(p, b, h, row) + c;
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = some ? o[2 * e] * inv : 0.f, y = some ? o[2 * e + 1] * inv : 0.f;
          if constexpr (std::is_same<T, __half>::value) w[e] = q4::pack_f16(x, y);
          else w[e] = q4::pack_bf16(x, y);
        }
        reinterpret_cast<uint4*>(at)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(at)[1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && dead != 0) raise(p.status, kTimeout);
  if (kLong && threadIdx.x == 0 && place >= 0) {  // all rows have theirs
    __threadfence();
    atomicExch(p.places + place, 0);
  }
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace kv8
}  // namespace tt
