// Products of many rows with a 4-bit matrix on the fifth-generation tensor
// cores (csrc/q4.cuh has the storage).
//
//   y[m,n]  = sum_k x[m,k] W^[n,k]        (rows of the tile: n, sum over k)
//   dx[m,k] = sum_n dy[m,n] W^[n,k]       (kTrans: rows k, sum over n)
//
// tcgen05.mma with fp16 operands: the matrix is decoded on the way into shared
// memory (operand A, 128 or 256 rows of a tile), the dense operand comes as
// fp16 through TMA (operand B, 32 to 256 tokens) and D = A B^T stays in TMEM.
// In fp16 nothing of a bf16-scaled matrix is lost: a code has at most 3
// significant bits (|c| <= 8), a bf16 scale 8, an fp16 number 11. Ranges are
// brought into fp16's by powers of two: each row n of W by e_n (its largest
// scale comes to 2^11..2^12), each row of the dense operand by f_m (to
// 2^13..2^14); they come off in the epilogue, or for the sum over n, e_n goes
// into dy. fp32 scales are taken as 8-bit terms and fp32 rows as two fp16
// terms, one pass over the sum for each pair of terms that matters.
//
// What bounds it: shared memory and the tensor cores for many tokens (256 x 256
// tiles, so that the L2 has to deliver only 40 bytes a clock and SM), the
// decoding for few (its warps then keep four blocks in flight each, and CTAs of
// a cluster share the sum when there are too few tiles for all SMs). bf16, 2048
// x 8192 x 8192: 223 us, 1.23 PFLOP/s, with 1.73 tiles an SM in two rounds;
// forward and backward of 2000 x 8192 x 4096 in fp16 271 us, 0.99 PFLOP/s.
// Roles: warps 0-15 decode (registers to swizzled shared memory, then, at the
// end, D to global memory), warp 16 issues the TMA loads, warp 17 the MMAs.
#pragma once
#include "ptx.cuh"
#include "ptx2sm.cuh"
#include "q4.cuh"

namespace tt {
namespace q4 {

constexpr int kDecodeWarps = 16;
constexpr int kGemmThreads = (kDecodeWarps + 2) * 32;
constexpr int kStageK = 64;  // terms of the sum in a stage: 128 bytes of fp16

struct Gemm {
  const uint4* packed;
  const void* scales;
  int scales_f32;          // fp32, else bf16
  const float* row_scale;  // 2^e_n
  const float* f;          // f_m, nullable: 1
  void* out;
  int type;                // of out
  long long ldo;
  int M, N, K, kblocks;
  int steps;               // 128-wide steps of the sum
  int passes;              // of the sum, one for each pair of terms:
  int scale_term[4], x_term[4];
  int tiles_m;
  int* err;
};

// kSums: sums leave TMEM in between (below).
template <int R, int MT, bool kSums>
struct GemmShape {
  static constexpr int kA = R * 128 * 128;  // bytes of operand A in a stage
  static constexpr int kB = MT * 128;
  static constexpr int kStageBytes = kA + kB;
  static constexpr int kStages = R == 2 ? 3 : MT == 256 ? 4 : MT == 128 ? 6 : 8;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static constexpr int kColumns = R * MT * (kSums ? 2 : 1);
  // half blocks that a decoding warp keeps in flight, for each of its R
  static constexpr int kDepth = R == 2 ? 2 : 4;
  // TMEM columns that a warp brings out at the end
  static constexpr int kOut = R * MT / 4 < 16 ? 16 : R * MT / 4;
  static_assert(kSmem <= 226 * 1024, "shared memory of an SM");
  static_assert(R == 2 || 128 * MT * 4 <= kStages * kStageBytes, "D fits where the stages were");
};

// Descriptors of operands in 128-byte swizzle are two words: the upper is the
// same for all (lines of eight rows 1 KB apart), the lower the address and, for
// row-major operands, the distance of their 64-row columns. The MMAs are issued
// by one lane of a warp that computes these words together, so that they stay
// in uniform registers: worked out by the lane alone they cost about 100 clocks
// an MMA, as much as a narrow one takes.
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo = 16) {
  return ((saddr >> 4) & 0x3FFFu) | (lbo >> 4) << 16;
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHigh)
      : "memory");
}
// fp16 operands, fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, int a_mn) {
  return (1u << 4) | ((uint32_t)a_mn << 15) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void store_out(const Gemm& p, long long i, float v) {
  if (p.type == kF32) static_cast<float*>(p.out)[i] = v;
  else if (p.type == kBF16) static_cast<__nv_bfloat16*>(p.out)[i] = from_f<__nv_bfloat16>(v);
  else static_cast<__half*>(p.out)[i] = from_f<__half>(v);
}
// The i-th 8-bit term of a scale.
__device__ __forceinline__ float scale_term(float s, int i) {
  const float a = __bfloat162float(__float2bfloat16_rn(s));
  if (i == 0) return a;
  const float r = s - a, b = __bfloat162float(__float2bfloat16_rn(r));
  return i == 1 ? b : r - b;
}

// The tensor cores cut an accumulator off to 24 bits at every addition: each of
// the K / 16 takes up to 2^-23 of the sum so far, to one side (measured where all
// terms have one sign: 1.1e-7 of the result a step for equal ones, 2.7e-8 for
// others; 1.2e-5 for fp32 rows, whose four passes make 470 of them of K = 1900).
// Results of 16 bits do not show it unless sums are very long. For those and for
// fp32 (kSums) D starts anew every kSumSteps steps of the sum, in the other half
// of TMEM, and the decoding warps add the finished half to fp32 registers: 16 cut
// additions at most, then rounded ones.
constexpr int kSumSteps = 2;

template <int R, int MT, int kGroups, bool kTrans, bool kSums>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_kernel(const __grid_constant__ CUtensorMap mapB, const Gemm p) {
  using S = GemmShape<R, MT, kSums>;
  static_assert(!kSums || R == 1, "D twice in TMEM");
  constexpr int kArrive = 8;  // decoding warps that fill a stage
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[S::kStages], empty[S::kStages], done, d_full[2], d_free[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int dead;  // a wait ran out
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = gridDim.x, rank = blockIdx.x;
  const long long tile = blockIdx.y + (long long)blockIdx.z * gridDim.y;
  const int m0 = (int)(tile % p.tiles_m) * MT;
  const long long row0 = tile / p.tiles_m * (R * 128);
  const long long rows = kTrans ? p.K : p.N;
  const bool active = row0 < rows;
  // this CTA's steps of the sum
  const int s0 = (int)((long long)p.steps * rank / splits), s1 = (int)((long long)p.steps * (rank + 1) / splits);
  const int count = active ? (s1 - s0) * p.passes : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], kArrive + 1);  // and the copies' arrival
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_free[i], kDecodeWarps);
    }
    fence_mbar_init();
    tma_prefetch_desc(&mapB);
    dead = 0;
  }
  if (warp == 17) {
    tmem_alloc(&tmem_slot, S::kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  bool ok = true;

  if (warp == 16) {
    if (lane == 0) {
      uint32_t it = 0;
      for (int i = 0, pass = 0, step = s0; i < count && ok; ++i) {
        for (int sub = 0; sub < 2; ++sub, ++it) {
          const int s = it % S::kStages;
          if (!mbar_wait(&empty[s], ((it / S::kStages) & 1u) ^ 1u, &dead, kDevTimeoutEmpty)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], S::kB);
          tma_load_3d(smem + s * S::kStageBytes + S::kA, &mapB, &full[s], step * 128 + sub * 64, m0,
                      p.x_term[pass]);
        }
        if (++step == s1) {
          step = s0;
          ++pass;
        }
      }
      for (uint32_t k = it > S::kStages ? it - S::kStages : 0; k < it; ++k)
        mbar_wait_drain(&full[k % S::kStages], (k / S::kStages) & 1u);
    }
    __syncwarp();
  } else if (warp == 17) {
    constexpr uint32_t idesc = idesc_f16(128, MT, kTrans ? 1 : 0);
    const uint32_t base = desc_low(smem_u32(smem), kTrans ? 8192 : 16), d0 = __shfl_sync(0xffffffffu, tmem, 0);
    uint32_t it = 0;
    for (; it < 2u * count; ++it) {
      const int s = it % S::kStages;
      const uint32_t ph = (it / S::kStages) & 1u;
      const uint32_t part = it / (2 * kSumSteps), of_part = it % (2 * kSumSteps);  // kSums
      if (kSums && of_part == 0 &&
          !__all_sync(0xffffffffu, mbar_wait(&d_free[part & 1], (part >> 1 & 1) ^ 1, &dead, kDevTimeoutAcc)))
        break;
      if (!__all_sync(0xffffffffu, mbar_wait(&full[s], ph, &dead, kDevTimeoutFull))) break;
      tc_fence_after();
      // sum-major A: 128-byte rows of 64 terms; row-major (kTrans): two columns
      // of 64 rows, 8 KB apart, one term to a 128-byte line
      const uint32_t a = base + s * (S::kStageBytes >> 4), b = a + (S::kA >> 4) - (kTrans ? (8192 - 16) << 12 : 0);
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < kStageK / 16; ++ks)
#pragma unroll
          for (int r = 0; r < R; ++r)
            mma_f16(d0 + (kSums ? (part & 1) * MT : r * MT), a + r * (16384 >> 4) + ks * ((kTrans ? 2048 : 32) >> 4), b + ks * (32 >> 4), idesc,
                    (kSums ? of_part : it) != 0 || ks != 0);
        mma_commit(&empty[s]);
        if (kSums && (of_part == 2 * kSumSteps - 1 || it + 1 == 2u * count)) mma_commit(&d_full[part & 1]);
      }
      __syncwarp();
    }
    if (elect_one()) {
      mma_commit(&done);
      mbar_wait_drain(&done, 0);
    }
    __syncwarp();
  } else {
    // A warp has row tile w8 of a step (or R of them) and the words 2 pair, 2
    // pair + 1 of its blocks: 64 columns. Those are a stage of the sum over k,
    // of which the step has two, or a column half of the sum over n, where
    // four row tiles make a stage.
    const int g = lane >> 2, t = lane & 3, odd = g & 1, w8 = warp & 7, pair = warp >> 3;
    const uint32_t sub = kTrans ? w8 >> 2 : pair;
    const long long rtiles = ((long long)p.N + kRows - 1) / kRows;
    constexpr int kScales = kGroups == 4 ? 2 : 1;  // of a word pair
    struct Piece {
      uint2 q[R][2];
      uint32_t s[R][2][kScales];
      uint32_t e[2];  // kTrans: 2^e_n of the two rows
    };
    Piece ring[S::kDepth];
    float down[R][2];  // 2^-e_n of this lane's rows
    auto inverse = [](float e) { return __uint_as_float(0x7f000000u - __float_as_uint(e)); };  // of a power of two
    if constexpr (!kTrans) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const long long n = row0 + r * 128 + w8 * 16 + g + 8 * h;
          down[r][h] = n < p.N ? inverse(__ldg(p.row_scale + n)) : 1.f;
        }
    }
    int next = s0;  // step to fetch
    // Everything is fetched from somewhere: what lies behind the last row tile
    // or block is dropped below, or never leaves the tile. One multiplication
    // an address: row tile (over n) or block (over k) times its bytes.
    const int size = p.scales_f32 ? 4 : 2;
    const char* at_q[R];
    const char* at_s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long blk = kTrans ? min(row0 / 128 + r, (long long)p.kblocks - 1)
                                   : min(row0 / 16 + r * 8 + w8, rtiles - 1) * p.kblocks;
      at_q[r] = reinterpret_cast<const char*>(p.packed) + blk * kBlockBytes + lane * 16 + pair * 8;
      at_s[r] = static_cast<const char*>(p.scales) + (blk * kGroups + pair * kGroups / 2) * kRows * size +
                (size == 4 ? g * 4 : (g & ~1) * 2);
    }
    auto fetch = [&](Piece& x) {
      const long long i = kTrans ? min(next * 8LL + w8, rtiles - 1) * p.kblocks : (long long)next;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const char* q = at_q[r] + i * kBlockBytes;
        const char* sc = at_s[r] + i * (kGroups * kRows * size);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          x.q[r][h] = ldg64(q + h * 512);
#pragma unroll
          for (int k = 0; k < kScales; ++k) x.s[r][h][k] = ldg32(sc + (k * kRows + 8 * h) * size);
        }
      }
      if constexpr (kTrans) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          x.e[h] = ldg32(p.row_scale + min(next * 128LL + w8 * 16 + g + 8 * h, (long long)p.N - 1));
      }
      if (++next == s1) next = s0;
    };
#pragma unroll
    for (int d = 0; d < S::kDepth; ++d) fetch(ring[d]);
    // Of D, a warp has lanes (its quarter of the rows) and a quarter of the
    // columns: of all 2 MT, rows 128 and up behind MT.
    const int quad = warp & 3, first = (warp >> 2) * S::kOut;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    float sum[kSums ? S::kOut : 1];
    int summed = 0;
    auto take = [&]() {  // the next part of the sum
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&d_full[summed & 1], summed >> 1 & 1, &dead, kDevTimeoutAcc));
      if (!ok) return;
      tc_fence_after();
      if (first < MT) {
#pragma unroll
        for (int c = 0; c < (kSums ? S::kOut : 0); c += 16) {
          float v[16];
          tmem_ld16(lanes + (summed & 1) * MT + first + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 16; ++k) sum[c + k] = summed == 0 ? v[k] : sum[c + k] + v[k];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&d_free[summed & 1]);
      ++summed;
    };
    int pass = 0, step = s0, term = p.scale_term[0];
    uint32_t it = sub;  // stage number
    // No way out of the loop but its head, and every turn fetches: the ring
    // then stays in its registers. (Leaving from the middle made copies of it,
    // which waited for the newest loads.)
    for (int i0 = 0; i0 < count; i0 += S::kDepth) {
#pragma unroll
      for (int d = 0; d < S::kDepth; ++d) {
        Piece& x = ring[d];
        const bool now = i0 + d < count && ok;
        if constexpr (kTrans) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < R; ++r) down[r][h] = inverse(__uint_as_float(x.e[h]));
        }
        uint4 v[R][2][2];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            __half2 sc[kScales];
#pragma unroll
            for (int k = 0; k < kScales; ++k) {
              // a row tile behind the last adds nothing, whatever was fetched for it
              const float f = !kTrans || step * 8LL + w8 < rtiles
                                  ? scale_value(x.s[r][h][k], p.scales_f32, odd) * down[r][h] : 0.f;
              sc[k] = __float2half2_rn(p.scales_f32 ? scale_term(f, term) : f);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // odd rows take the pair's words the other way round: eight
              // lanes then meet all 32 banks
              const uint32_t wd = (e == odd) ? x.q[r][h].x : x.q[r][h].y;
              const __half2 sh = kScales == 1 ? sc[0] : (e == odd ? sc[0] : sc[kScales - 1]);
              uint32_t y[4];
#pragma unroll
              for (int j = 0; j < 4; j += 2) {
                uint32_t lo, hi;
                decode_two_pairs(wd >> (4 * j), lo, hi);
                const __half2 a = __hmul2(reinterpret_cast<const __half2&>(lo), sh);
                const __half2 b = __hmul2(reinterpret_cast<const __half2&>(hi), sh);
                y[j] = reinterpret_cast<const uint32_t&>(a);
                y[j + 1] = reinterpret_cast<const uint32_t&>(b);
              }
              v[r][h][e] = make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
        fetch(x);
        if (now) {
        const int s = it % S::kStages;
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ((it / S::kStages) & 1u) ^ 1u, &dead, kDevTimeoutEmpty));
        const uint32_t base = smem_u32(smem + s * S::kStageBytes);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t n = kTrans ? (w8 & 3) * 16 + g + 8 * h : r * 128 + w8 * 16 + g + 8 * h;
              const uint32_t chunk = (uint32_t)((e ^ odd) * 4 + t);
              const uint32_t at = base + (kTrans ? (2 * r + pair) * 8192 : 0) + n * 128 + ((chunk ^ (n & 7)) << 4);
              asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[r][h][e].x), "r"(v[r][h][e].y),
                           "r"(v[r][h][e].z), "r"(v[r][h][e].w)
                           : "memory");
            }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
        }
        if constexpr (kSums)  // one part behind
          if (now && (i0 + d) % kSumSteps == kSumSteps - 1 && i0 + d >= 2 * kSumSteps - 1) take();
        it += 2;
        if (++step == s1) {
          step = s0;
          ++pass;
          if (pass < p.passes) term = p.scale_term[pass];
        }
      }
    }
    if constexpr (kSums)
      while (ok && summed * kSumSteps < count) take();
    // D: lanes are rows of the tile, columns are tokens. Where a wait ran out,
    // here or in an earlier call that nobody has looked at yet, it is NaN.
    ok = *(volatile int*)p.err == 0 && ok;
    ok = mbar_wait(&done, 0, &dead, kDevTimeoutAcc) && ok;
    ok = __all_sync(0xffffffffu, ok && *(volatile int*)&dead == 0);
    tc_fence_after();
    if (active) {
      const int half = R == 2 ? first / MT : 0;
      const long long row = row0 + half * 128 + quad * 32 + lane;
      const int c0 = first - half * MT;
      const float up = !kTrans && row < rows ? __ldg(p.row_scale + row) : 1.f;
      float* dsm = reinterpret_cast<float*>(smem);
      auto bring = [&](int c, const float (&v)[16]) {
        if (splits > 1) {
#pragma unroll
          for (int k = 0; k < 16; ++k) dsm[(c + k) * 128 + quad * 32 + lane] = v[k];
        } else if (row < rows) {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int m = m0 + c + k;
            if (m < p.M)
              store_out(p, m * p.ldo + row, v[k] * up * (p.f ? __ldg(p.f + m) : 1.f));
          }
        }
      };
      const int c1 = first < R * MT ? c0 + S::kOut : c0;
      float v[16];
      if (!ok) {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = __int_as_float(0x7fffffff);
        for (int c = c0; c < c1 && m0 + c < p.M; c += 16) bring(c, v);
      } else if constexpr (kSums) {
#pragma unroll
        for (int j = 0; j < S::kOut; j += 16) {
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = sum[j + k];
          if (c0 < c1 && m0 + c0 + j < p.M) bring(c0 + j, v);
        }
      } else {
        for (int c = c0; c < c1 && m0 + c < p.M; c += 16) {
          tmem_ld16(lanes + half * MT + c, v);
          tmem_ld_wait();
          bring(c, v);
        }
      }
    }
  }
  if (splits > 1) {  // the CTAs' parts, added in rank order, a share of the tokens each
    cluster_sync();
    if (R == 1 && active && threadIdx.x < 256) {
      const int r = threadIdx.x & 127;
      const long long row = row0 + r;
      const float up = !kTrans && row < rows ? __ldg(p.row_scale + row) : 1.f;
      const uint32_t base = smem_u32(smem);
      for (int c = rank + splits * (threadIdx.x >> 7); c < MT && m0 + c < p.M; c += 2 * splits) {
        float v = 0.f;
        for (int k = 0; k < splits; ++k) {
          float w;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(w) : "r"(mapa(base + (c * 128 + r) * 4, k)));
          v += w;
        }
        const int m = m0 + c;
        if (row < rows)
          store_out(p, m * p.ldo + row, v * up * (p.f ? __ldg(p.f + m) : 1.f));
      }
    }
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && dead != 0) atomicCAS(p.err, 0, dead);
  if (warp == 17) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kColumns);
  }
}

// 2^e_n of each row: the exponent that brings its largest finite |s| to
// 2^11 .. 2^12 when divided by. A row of zeros gets the smallest: over n the
// power goes into dy, whose largest product sets the range for all others, and
// dy of such a row (but for an infinity or NaN) counts for nothing.
template <typename ST>
__global__ void row_scale_kernel(const ST* __restrict__ scales, int N, int kblocks, int gpb,
                                 float* __restrict__ out) {
  // a warp a row tile: lanes 0-15 and 16-31 are its rows, taking turns
  const long long rt = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  const long long rtiles = ((long long)N + kRows - 1) / kRows;
  if (rt >= rtiles) return;
  const long long lines = (long long)kblocks * gpb;
  const ST* at = scales + rt * lines * kRows;
  uint32_t top = 0;
  for (long long i = lane; i < lines * kRows; i += 32) {
    const uint32_t b = __float_as_uint(fabsf(to_f(at[i])));
    if (b < 0x7f800000u) top = max(top, b);
  }
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
  int e = (int)(top >> 23) - 11;  // biased exponent of 2^e
  e = e < 1 ? 1 : e > 253 ? 253 : e;
  const long long n = rt * kRows + (lane & 15);
  if (lane < 16 && n < N) out[n] = __uint_as_float((uint32_t)e << 23);
}

// Rows of the dense operand as fp16: x 2^e (e by column, or none), times the
// power of two that brings the row's largest finite value to 2^13 .. 2^14,
// rounded (kTerms 1) or as two terms; zeros behind the row's end. f gets the
// power's reciprocal. `finite`: one more copy of the first term, without
// infinities and NaN, for the passes of a scale's smaller terms (an infinity
// enters the sum once).
template <typename XT, int kTerms>
__global__ void __launch_bounds__(256)
convert_kernel(const XT* __restrict__ x, long long ldx, const float* __restrict__ col, int M, int C, int Cp, int wide,
               __half* __restrict__ out, float* __restrict__ f, int finite) {
  __shared__ uint32_t tops[8];
  const int m = blockIdx.x;
  const XT* row = x + m * ldx;
  // eight neighbouring values of the row, zeros behind its end
  auto eight = [&](int i, float (&v)[8]) {
    constexpr int kPer = 16 / sizeof(XT);
    if (wide && i + 8 <= C) {
#pragma unroll
      for (int j = 0; j < 8 / kPer; ++j) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + i) + j);
        const XT* e = reinterpret_cast<const XT*>(&u);
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[j * kPer + k] = to_f(e[k]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i + j < C ? to_f(__ldg(row + i + j)) : 0.f;
    }
    if (col) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= i + j < C ? __ldg(col + i + j) : 1.f;
    }
  };
  uint32_t top = 0;
#pragma unroll 2
  for (int i = threadIdx.x * 8; i < C; i += 2048) {
    float v[8];
    eight(i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(fabsf(v[j]));
      top = max(top, b < 0x7f800000u ? b : 0u);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = max(top, tops[w]);
  int e = (int)(top >> 23);
  e = e < 14 ? 14 : e;
  const float up = __uint_as_float((uint32_t)(267 - e) << 23);  // 2^(140 - e)
  if (threadIdx.x == 0) f[m] = __uint_as_float((uint32_t)(e - 13) << 23);
  __half* hi = out + (long long)m * Cp;
  const long long plane = (long long)M * Cp;
  auto put = [&](__half* at, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(at) =
        make_uint4(pack_f16(v[0], v[1]), pack_f16(v[2], v[3]), pack_f16(v[4], v[5]), pack_f16(v[6], v[7]));
  };
#pragma unroll 2
  for (int i = threadIdx.x * 8; i < Cp; i += 2048) {
    float v[8];
    eight(i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= up;
    put(hi + i, v);
    if (kTerms == 2) {
      float lo[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) lo[j] = isfinite(v[j]) ? v[j] - __half2float(__float2half_rn(v[j])) : 0.f;
      put(hi + plane + i, lo);
    }
    if (finite) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = isfinite(v[j]) ? v[j] : 0.f;
      put(hi + kTerms * plane + i, v);
    }
  }
}

}  // namespace q4
}  // namespace tt
