// 4-bit matrices with group scales: packing, quantisation, decoding, and the
// products with few rows (csrc/q4.cuh describes the storage).
//
//   y[m,n]  = sum_k x[m,k] s[n,g(k)] c[n,k]
//   dx[m,k] = sum_n dy[m,n] s[n,g(k)] c[n,k]
//
// Both products with few rows read the matrix once (4.1 bits a weight). What
// bounds them is not that yet but the instructions that decode it and the wait
// for the first bytes. The codes are exact in bf16 and fp16, so the products
// run on mma.sync tensor-core fragments decoded in registers and accumulate
// in fp32; tcgen05 would want the decoded matrix in shared memory first,
// which costs more than it saves while the rows fit one fragment.
#include <cooperative_groups.h>

#include "common.cuh"
#include "q4.cuh"
#include "q4_host.cuh"

namespace tt {
namespace q4 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8;
constexpr int kMaxCluster = 8;
// Up to so many rows the products run here, above in csrc/q4_gemm.cuh. Measured
// on both sides with 16384 x 8192 and 4096 x 4096, in us: over k, 32 rows of
// bf16 40 here and 44 there, 16 rows of fp32 190 and 28 here, 101 and 20 there;
// over n, 16 rows of bf16 63 and 30 here, 60 and 16 there, of fp32 68 and 30
// here, 122 and 23 there.
int few_rows(int type, bool transposed) { return transposed ? (type == kF32 ? 16 : 8) : type == kF32 ? 8 : 32; }

// ------------------------------------------------------- packing and decoding

// One warp a block of 16 x 128. kFrom: the codes are given (pack) or made from
// W (quantise: s = amax / 7 rounded to the scale's type, c = rint(w / s)).
template <typename WT, typename ST>
__global__ void quantize_kernel(const WT* __restrict__ W, long long ldw, int N, int K, int group,
                                uint4* __restrict__ packed, ST* __restrict__ scales,
                                long long blocks, int kblocks) {
  const long long blk = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (blk >= blocks) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long rt = blk / kblocks;
  const int kb = (int)(blk % kblocks);
  const int words = group / 32, gpb = 4 / words;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long long row = rt * kRows + g + 8 * h;
    float v[4][8];
    uint32_t top[4];  // largest |w| by its bits, whose order puts infinities and NaN on top
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      top[w] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const long long k = (long long)kb * kCols + 32 * w + 8 * t + i;
        v[w][i] = row < N && k < K ? to_f(W[row * ldw + k]) : 0.f;
        top[w] = max(top[w], __float_as_uint(fabsf(v[w][i])));
      }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) top[w] = max(top[w], __shfl_xor_sync(0xffffffffu, top[w], o));
    uint32_t out[4];
#pragma unroll
    for (int gi = 0; gi < 4; ++gi) {
      if (gi >= gpb) break;
      uint32_t bits = 0;
      for (int w = gi * words; w < (gi + 1) * words; ++w) bits = max(bits, top[w]);
      const float m = bits >= 0x7f800000u ? __int_as_float(0x7fffffff) : __uint_as_float(bits);
      const ST st = from_f<ST>(__fdiv_rn(m, 7.f));
      const float s = to_f(st);
      if (t == 0) scales[(blk * gpb + gi) * kRows + g + 8 * h] = st;
      for (int w = gi * words; w < (gi + 1) * words; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float c = s > 0.f ? rintf(__fdiv_rn(v[w][i], s)) : 0.f;
          c = fminf(fmaxf(c, -8.f), 7.f);
          word |= (uint32_t)((int)c + 8) << (4 * (i / 2 + 4 * (i & 1)));
        }
        out[w] = word;
      }
    }
    packed[blk * 64 + h * 32 + lane] = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

template <typename ST>
__global__ void pack_kernel(const signed char* __restrict__ codes, const ST* __restrict__ in_scales,
                            int N, int K, int group, uint4* __restrict__ packed,
                            ST* __restrict__ scales, long long blocks, int kblocks) {
  const long long blk = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (blk >= blocks) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long rt = blk / kblocks;
  const int kb = (int)(blk % kblocks);
  const int gpb = kCols / group;
  const long long groups = ((long long)K + group - 1) / group;
  const bool wide = K % 8 == 0 && (reinterpret_cast<uintptr_t>(codes) & 7u) == 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long long row = rt * kRows + g + 8 * h;
    uint32_t out[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const long long k0 = (long long)kb * kCols + 32 * w + 8 * t;
      signed char c[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (row < N && wide && k0 < K) {
        *reinterpret_cast<uint2*>(c) = *reinterpret_cast<const uint2*>(codes + row * K + k0);
      } else if (row < N) {
        for (int i = 0; i < 8; ++i)
          if (k0 + i < K) c[i] = codes[row * K + k0 + i];
      }
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        word |= (uint32_t)((c[i] + 8) & 15) << (4 * (i / 2 + 4 * (i & 1)));
      out[w] = word;
    }
    packed[blk * 64 + h * 32 + lane] = make_uint4(out[0], out[1], out[2], out[3]);
    if (t < gpb) {
      const long long gi = (long long)kb * gpb + t;
      scales[(blk * gpb + t) * kRows + g + 8 * h] =
          row < N && gi < groups ? in_scales[row * groups + gi] : from_f<ST>(0.f);
    }
  }
}

template <typename OT, typename ST>
__global__ void dequantize_kernel(const uint4* __restrict__ packed, const ST* __restrict__ scales,
                                  int N, int K, int group, OT* __restrict__ out, long long blocks,
                                  int kblocks) {
  const long long blk = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (blk >= blocks) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long rt = blk / kblocks;
  const int kb = (int)(blk % kblocks);
  const int gpb = kCols / group;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long long row = rt * kRows + g + 8 * h;
    if (row >= N) continue;
    const uint4 q = packed[blk * 64 + h * 32 + lane];
    const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float s = to_f(scales[(blk * gpb + w * gpb / 4) * kRows + g + 8 * h]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const long long k = (long long)kb * kCols + 32 * w + 8 * t + i;
        const int c = (int)((word[w] >> (4 * (i / 2 + 4 * (i & 1)))) & 15u) - 8;
        if (k < K) out[row * K + k] = from_f<OT>(s * (float)c);
      }
    }
  }
}

// ------------------------------------------------------------------ operands

// Eight neighbouring values as pairs for kTerms fragments. `wide`: all are
// there and 16-byte aligned; else the first `left` are, and zeros follow.
template <typename XT, int kTerms>
__device__ __forceinline__ void load_eight(const XT* __restrict__ at, int left, bool wide, uint32_t (&out)[kTerms][4]) {
  if constexpr (sizeof(XT) == 2) {
    if (wide) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(at));
      out[0][0] = v.x; out[0][1] = v.y; out[0][2] = v.z; out[0][3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t lo = 0, hi = 0;
        if (2 * j < left) lo = __ldg(reinterpret_cast<const unsigned short*>(at) + 2 * j);
        if (2 * j + 1 < left) hi = __ldg(reinterpret_cast<const unsigned short*>(at) + 2 * j + 1);
        out[0][j] = lo | hi << 16;
      }
    }
  } else {
    float f[8];
    if (wide) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(at)), b = __ldg(reinterpret_cast<const float4*>(at) + 1);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = i < left ? __ldg(at + i) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t p[kTerms];
      split_bf16<kTerms>(f[2 * j], f[2 * j + 1], p);
#pragma unroll
      for (int i = 0; i < kTerms; ++i) out[i][j] = p[i];
    }
  }
}

// ------------------------------------------------------------ y = x W^T, few rows

// Up to eight tokens. A CTA owns 16 rows of W; its warps take the row tile's
// blocks in turn, and the CTAs of a cluster (blockIdx.x is the rank) share
// them, so that a short matrix still fills the GPU. Each group of k gets a
// fragment of its own, which is scaled in fp32 when the group ends. The parts
// are added in a fixed order: warps through shared memory, CTAs through the
// cluster's. bf16, one row: 4096 x 4096 5 us (1.6 TB/s of matrix, mostly the
// launch and the first wait), 16384 x 8192 25 us (2.8 TB/s: 187 instructions a
// block of 1 KB fill half of the issue slots, and waits for memory the rest).
template <typename XT, typename ST, int kGroups>
__global__ void __launch_bounds__(kWarps * 32, sizeof(XT) == 2 ? 3 : 1)
matvec_kernel(const XT* __restrict__ x, long long ldx, const uint4* __restrict__ packed,
              const ST* __restrict__ scales, int M, int N, int K, int kblocks, int wide,
              XT* __restrict__ y, long long ldy) {
  constexpr bool kHalf = sizeof(XT) == 2 && !std::is_same<XT, __nv_bfloat16>::value;
  constexpr int kTerms = sizeof(XT) == 2 ? 1 : 3;
  constexpr int kOut = kRows * 8;
  __shared__ float part[kWarps * kOut];
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x / 32, warps = blockDim.x / 32, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int splits = gridDim.x;
  const long long rt = blockIdx.y + (long long)blockIdx.z * gridDim.y;
  const long long rtiles = ((long long)N + kRows - 1) / kRows;
  const bool active = rt < rtiles;

  float acc[4] = {0.f, 0.f, 0.f, 0.f};

  if (active) {
    // a token that is not there reads another's values: its column is dropped
    const XT* xr = x + (long long)min(g, M - 1) * ldx + 8 * t;
    const int whole = wide ? K / kCols : 0;  // blocks whose 128 columns can be read as they stand
    // A ring of blocks in registers: codes, scales and the tokens' values are
    // asked for kDepth blocks ahead.
    constexpr int kDepth = 2;
    constexpr bool kF32Scale = sizeof(ST) == 4;
    struct Piece {
      uint4 qa, qb;
      uint32_t s[kGroups][2];
    };
    Piece ring[kDepth];
    const int stride = splits * warps;
    int next = blockIdx.x * warps + warp;
    auto fetch = [&](Piece& f) {  // behind the last block: the last again, for nothing
      const long long blk = rt * kblocks + min(next, kblocks - 1);
      f.qa = ldg128(packed + blk * 64 + lane);
      f.qb = ldg128(packed + blk * 64 + 32 + lane);
#pragma unroll
      for (int gi = 0; gi < kGroups; ++gi) {
        f.s[gi][0] = scale_word(scales, kF32Scale, (blk * kGroups + gi) * kRows + g);
        f.s[gi][1] = scale_word(scales, kF32Scale, (blk * kGroups + gi) * kRows + g + 8);
      }
      next += stride;
    };
#pragma unroll
    for (int d = 0; d < kDepth; ++d) fetch(ring[d]);
    for (int kb0 = blockIdx.x * warps + warp; kb0 < kblocks; kb0 += stride * kDepth) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        // past the end the last block is fetched again, and counts for nothing
        const int kb = min(kb0 + d * stride, kblocks - 1);
        const bool on = kb0 + d * stride < kblocks;
        uint32_t xp[4][kTerms][4];
#pragma unroll
        for (int w = 0; w < 4; ++w)
          load_eight<XT, kTerms>(xr + (long long)kb * kCols + 32 * w, K - kb * kCols - 32 * w - 8 * t, kb < whole,
                                 xp[w]);
        const Piece f = ring[d];
        fetch(ring[d]);
        const uint32_t wa[4] = {f.qa.x, f.qa.y, f.qa.z, f.qa.w}, wb[4] = {f.qb.x, f.qb.y, f.qb.z, f.qb.w};
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = gi * 4 / kGroups; w < (gi + 1) * 4 / kGroups; ++w)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t a0, a1, a2, a3;
              decode_four<kHalf>(wa[w] >> (8 * half), a0, a2);
              decode_four<kHalf>(wb[w] >> (8 * half), a1, a3);
#pragma unroll
              for (int i = 0; i < kTerms; ++i)
                mma16816<kHalf>(c, a0, a1, a2, a3, xp[w][i][2 * half], xp[w][i][2 * half + 1]);
            }
          const float s0 = scale_value(f.s[gi][0], kF32Scale, g & 1), s1 = scale_value(f.s[gi][1], kF32Scale, g & 1);
          if (on) {
            acc[0] += s0 * c[0];
            acc[1] += s0 * c[1];
            acc[2] += s1 * c[2];
            acc[3] += s1 * c[3];
          }
        }
      }
    }
  }
  // part[warp][token][row]
  float* mine = part + warp * kOut;
  mine[2 * t * kRows + g] = acc[0];
  mine[(2 * t + 1) * kRows + g] = acc[1];
  mine[2 * t * kRows + g + 8] = acc[2];
  mine[(2 * t + 1) * kRows + g + 8] = acc[3];
  __syncthreads();
  for (int o = threadIdx.x; o < kOut; o += blockDim.x) {
    float v = part[o];
    for (int w = 1; w < warps; ++w) v += part[w * kOut + o];
    part[o] = v;
  }
  if (splits > 1) {
    cluster.sync();
    if (blockIdx.x == 0) {
      for (int o = threadIdx.x; o < kOut; o += blockDim.x) {
        float v = part[o];
        for (int r = 1; r < splits; ++r) v += cluster.map_shared_rank(part, r)[o];
        part[o] = v;
      }
    }
    cluster.sync();
  } else {
    __syncthreads();
  }
  if (blockIdx.x == 0 && active) {
    for (int o = threadIdx.x; o < kOut; o += blockDim.x) {
      const long long m = o / kRows, n = rt * kRows + o % kRows;
      if (m < M && n < N) y[m * ldy + n] = from_f<XT>(part[o]);
    }
  }
}

// A value from its bits (16-bit types in the low half).
template <typename T>
__device__ __forceinline__ float value_of(uint32_t bits) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)bits));
  else return __uint_as_float(bits << 16);
}

// ------------------------------------------------------------ dx = dy W, few rows

// A CTA owns 128 columns of W and 8 kTiles tokens; the rows of W are shared
// among its warps and the CTAs of its cluster. Here the scale varies along the
// sum, so it goes into the other operand: dy s is split into bf16 terms (two
// for 16-bit types: 2^-16 of each product, against 2^-9 or 2^-12 for the
// result's own rounding; three for fp32). A fragment of W takes the columns
// k = 32 w + 8 (c / 2) + 2 j + c % 2 of a block, c = 0 .. 7, for two j, so that
// all its columns share a group. The tensor cores cut off at every addition,
// which a long sum in fp32 shows (2.4e-6 of the result for 14000 rows): there
// the fragments are emptied into rounded sums every four row tiles. bf16, one row: 4096 x 4096 9.6 us, 16384 x
// 8192 35 us (2.0 TB/s): decoding and the doubled products bound it.
template <typename XT, typename ST, int kTiles, int kGroups>
__global__ void __launch_bounds__(kWarps * 32, kTiles == 1 ? 2 : 1)
matvec_t_kernel(const XT* __restrict__ dy, long long lddy, const uint4* __restrict__ packed,
                const ST* __restrict__ scales, int M, int N, int K, int kblocks,
                XT* __restrict__ dx, long long lddx) {
  constexpr int kTerms = sizeof(XT) == 2 ? 2 : 3;
  constexpr int kTok = 8 * kTiles, kRow = kCols + 4;  // a row's floats in shared memory
  extern __shared__ float tpart[];  // [warp][token][kRow]
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x / 32, warps = blockDim.x / 32, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int splits = gridDim.x;
  const long long tile = blockIdx.y + (long long)blockIdx.z * gridDim.y;
  const long long mtiles = ((long long)M + kTok - 1) / kTok;
  const bool active = tile < (long long)kblocks * mtiles;
  const int kb = active ? (int)(tile % kblocks) : 0;
  const long long m0 = active ? tile / kblocks * kTok : 0;
  const int rtiles = (int)(((long long)N + kRows - 1) / kRows);

  float acc[kTiles][8][4];
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][i][e] = 0.f;

  if (active) {
    constexpr bool kF32Scale = sizeof(ST) == 4;
    struct Piece {
      uint4 q[4];                // rows 2t, 2t+1, 8+2t, 9+2t; the words of t' = g / 2
      uint32_t d[kTiles][4];     // token g, those rows: bits of dy
      uint32_t s[kGroups][kF32Scale ? 4 : 2];  // bf16: two neighbours in a word
    };
    constexpr int kDepth = 2;
    Piece ring[kDepth];
    const int stride = splits * warps;
    int next = blockIdx.x * warps + warp;
    const XT* row[kTiles];  // a token that is not there reads another's: its column is dropped
#pragma unroll
    for (int j = 0; j < kTiles; ++j) row[j] = dy + min(m0 + 8 * j + g, (long long)M - 1) * lddy;
    const uint4* at_q = packed + (long long)kb * 64 + 2 * t * 4 + (g >> 1);
    auto fetch = [&](Piece& f) {  // behind the last row tile: the last again, for nothing
      const int rt = min(next, rtiles - 1);
      const uint4* q = at_q + (long long)rt * kblocks * 64;
#pragma unroll
      for (int r = 0; r < 4; ++r) f.q[r] = ldg128(q + (r >> 1) * 32 + (r & 1) * 4);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = min(rt * kRows + (r >> 1) * 8 + 2 * t + (r & 1), N - 1);
#pragma unroll
        for (int j = 0; j < kTiles; ++j) f.d[j][r] = sizeof(XT) == 4 ? ldg32(row[j] + n) : ldg16(row[j] + n);
      }
#pragma unroll
      for (int gi = 0; gi < kGroups; ++gi) {
        const ST* s = scales + (((long long)rt * kblocks + kb) * kGroups + gi) * kRows + 2 * t;
        if constexpr (kF32Scale) {
#pragma unroll
          for (int r = 0; r < 4; ++r) f.s[gi][r] = ldg32(s + (r >> 1) * 8 + (r & 1));
        } else {
          f.s[gi][0] = ldg32(s);
          f.s[gi][1] = ldg32(s + 8);
        }
      }
      next += stride;
    };
#pragma unroll
    for (int d = 0; d < kDepth; ++d) fetch(ring[d]);
    float whole[kTerms == 3 ? kTiles : 1][8][4] = {};
    int turn = 0;
    for (int rt0 = blockIdx.x * warps + warp; rt0 < rtiles; rt0 += stride * kDepth) {
      if constexpr (kTerms == 3) {
        if (turn++ & 1) {
#pragma unroll
          for (int j = 0; j < kTiles; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                whole[j][i][e] += acc[j][i][e];
                acc[j][i][e] = 0.f;
              }
        }
      }
#pragma unroll
      for (int dd = 0; dd < kDepth; ++dd) {
        const int rt = rt0 + dd * stride;  // behind the last: dy counts as zero, and the scale too
        const Piece f = ring[dd];
        fetch(ring[dd]);
        float d[kTiles][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = rt * kRows + (r >> 1) * 8 + 2 * t + (r & 1) < N;
#pragma unroll
          for (int j = 0; j < kTiles; ++j) d[j][r] = in ? value_of<XT>(f.d[j][r]) : 0.f;
        }
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) {
          float s[4];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[r] = rt >= rtiles ? 0.f : kF32Scale ? __uint_as_float(f.s[gi][r]) : scale_value(f.s[gi][r >> 1], false, r & 1);
          uint32_t b[kTiles][2][kTerms];
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            split_bf16<kTerms>(d[j][0] * s[0], d[j][1] * s[1], b[j][0]);
            split_bf16<kTerms>(d[j][2] * s[2], d[j][3] * s[3], b[j][1]);
          }
#pragma unroll
          for (int w = gi * 4 / kGroups; w < (gi + 1) * 4 / kGroups; ++w) {
            const uint32_t sel = g & 1 ? 0x7632 : 0x5410;
            auto word = [&](int r) { return w == 0 ? f.q[r].x : w == 1 ? f.q[r].y : w == 2 ? f.q[r].z : f.q[r].w; };
            const uint32_t lo = __byte_perm(word(0), word(1), sel), hi = __byte_perm(word(2), word(3), sel);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t a0 = decode_pair<false>(lo >> (8 * i)), a1 = decode_pair<false>(lo >> (8 * i + 4));
              const uint32_t a2 = decode_pair<false>(hi >> (8 * i)), a3 = decode_pair<false>(hi >> (8 * i + 4));
#pragma unroll
              for (int j = 0; j < kTiles; ++j)
#pragma unroll
                for (int k = 0; k < kTerms; ++k)
                  mma16816<false>(acc[j][2 * w + i], a0, a1, a2, a3, b[j][0][k], b[j][1][k]);
            }
          }
        }
      }
    }
    if constexpr (kTerms == 3) {
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][i][e] += whole[j][i][e];
    }
  }
  // acc[j][2 w + i]: columns 32 w + 8 (g / 2) + 4 i + g % 2, and 2 on, tokens 8 j + 2 t, 2 t + 1
  float* mine = tpart + warp * kTok * kRow;
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mine[(8 * j + 2 * t + (e & 1)) * kRow + 32 * (i >> 1) + 8 * (g >> 1) + 4 * (i & 1) + (g & 1) + 2 * (e >> 1)] =
            acc[j][i][e];
  __syncthreads();
  constexpr int kOut = kTok * kCols;
  for (int o = threadIdx.x; o < kOut; o += blockDim.x) {
    const int at = o / kCols * kRow + o % kCols;
    float v = tpart[at];
    for (int w = 1; w < warps; ++w) v += tpart[w * kTok * kRow + at];
    tpart[at] = v;
  }
  if (splits > 1) {
    cluster.sync();
    // every rank adds a share of the outputs, in rank order, and keeps it to itself
    if (active) {
      for (int o = threadIdx.x + blockIdx.x * blockDim.x; o < kOut; o += splits * blockDim.x) {
        const int at = o / kCols * kRow + o % kCols;
        float v = cluster.map_shared_rank(tpart, 0)[at];
        for (int r = 1; r < splits; ++r) v += cluster.map_shared_rank(tpart, r)[at];
        const long long m = m0 + o / kCols, k = (long long)kb * kCols + o % kCols;
        if (m < M && k < K) dx[m * lddx + k] = from_f<XT>(v);
      }
    }
    cluster.sync();
  } else {
    __syncthreads();
    if (active) {
      for (int o = threadIdx.x; o < kOut; o += blockDim.x) {
        const long long m = m0 + o / kCols, k = (long long)kb * kCols + o % kCols;
        if (m < M && k < K) dx[m * lddx + k] = from_f<XT>(tpart[o / kCols * kRow + o % kCols]);
      }
    }
  }
}

// ------------------------------------------------- y = x W^T, up to 32 rows

// As the first product, for 16-bit types and 9 to 32 tokens. There the tokens'
// values are what a warp reads most of, so a CTA takes 128 rows of W, one row
// tile a warp, and all its warps share the tokens' values from shared memory:
// four blocks of k a stage, filled by cp.async one stage ahead, rows 64 bytes
// off each other's banks. The CTAs of a cluster share the sum over k.
// 32 x 16384 x 8192 in bf16 takes 40 us (1.7 TB/s of matrix): about 270
// instructions a block and row tile, 41% of the time on the products alone (17
// us at the least). tcgen05 with the matrix decoded into shared memory takes 44
// (csrc/q4_gemm.cuh); CTAs of seven warps, which would fill the SMs evenly,
// took 43.
constexpr int kMidBlocks = 4;                                // of k in a stage
constexpr int kMidRow = kMidBlocks * kCols * 2 + 64;         // bytes of a token's row there
constexpr int kMidStages = 2;

template <int kTiles>
constexpr int mid_smem() { return kMidStages * 8 * kTiles * kMidRow; }

template <typename XT, typename ST, int kTiles, int kGroups>
__global__ void __launch_bounds__(kWarps * 32, 2)
mid_kernel(const XT* __restrict__ x, long long ldx, const uint4* __restrict__ packed, const ST* __restrict__ scales,
           int M, int N, int K, int kblocks, int wide, XT* __restrict__ y, long long ldy) {
  constexpr bool kHalf = !std::is_same<XT, __nv_bfloat16>::value;
  constexpr bool kF32Scale = sizeof(ST) == 4;
  constexpr int kTok = 8 * kTiles;
  extern __shared__ __align__(16) unsigned char msm[];
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int splits = gridDim.x;
  const long long group_of = blockIdx.y + (long long)blockIdx.z * gridDim.y;
  const int rtiles = (int)(((long long)N + kRows - 1) / kRows);
  const bool active = group_of * kWarps < rtiles;
  const int rt = (int)min(group_of * kWarps + warp, (long long)rtiles - 1);  // behind the last: dropped at the end
  const int b0 = (int)((long long)kblocks * blockIdx.x / splits), b1 = (int)((long long)kblocks * (blockIdx.x + 1) / splits);
  const int stages = active ? (b1 - b0 + kMidBlocks - 1) / kMidBlocks : 0;

  // a stage's values: token by token, 16 bytes a thread; zeros where there are none
  auto fill = [&](int s) {
    unsigned char* to = msm + (s % kMidStages) * kTok * kMidRow;
    const int k0 = (b0 + s * kMidBlocks) * kCols;
    for (int i = threadIdx.x; i < kTok * kMidBlocks * 16; i += kWarps * 32) {
      const int m = i / (kMidBlocks * 16), c = i % (kMidBlocks * 16), k = k0 + 8 * c;
      unsigned char* at = to + m * kMidRow + 16 * c;
      const XT* from = x + (long long)min(m, M - 1) * ldx + k;
      if (wide && k + 8 <= K) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(at)), "l"(from)
                     : "memory");
      } else {
        uint32_t v[1][4];
        load_eight<XT, 1>(from, K - k, false, v);
        *reinterpret_cast<uint4*>(at) = make_uint4(v[0][0], v[0][1], v[0][2], v[0][3]);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  float acc[kTiles][4];
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
  struct Piece {
    uint4 qa, qb;
    uint32_t s[kGroups][2];
  };
  constexpr int kDepth = kMidBlocks;
  Piece ring[kDepth];
  int next = b0;
  const uint4* at_q = packed + (long long)rt * kblocks * 64 + lane;
  auto fetch = [&](Piece& f) {
    const int kb = min(next, b1 - 1);
    f.qa = ldg128(at_q + (long long)kb * 64);
    f.qb = ldg128(at_q + (long long)kb * 64 + 32);
#pragma unroll
    for (int gi = 0; gi < kGroups; ++gi) {
      f.s[gi][0] = scale_word(scales, kF32Scale, (((long long)rt * kblocks + kb) * kGroups + gi) * kRows + g);
      f.s[gi][1] = scale_word(scales, kF32Scale, (((long long)rt * kblocks + kb) * kGroups + gi) * kRows + g + 8);
    }
    ++next;
  };
  if (stages > 0) {
    fill(0);
#pragma unroll
    for (int d = 0; d < kDepth; ++d) fetch(ring[d]);
  }
  for (int s = 0; s < stages; ++s) {
    if (s + 1 < stages) fill(s + 1);
    else asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    const unsigned char* from = msm + (s % kMidStages) * kTok * kMidRow + g * kMidRow + t * 16;
#pragma unroll
    for (int i = 0; i < kMidBlocks; ++i) {
      const bool on = b0 + s * kMidBlocks + i < b1;  // else the last block again, for nothing
      const Piece f = ring[i % kDepth];
      fetch(ring[i % kDepth]);
      const uint32_t wa[4] = {f.qa.x, f.qa.y, f.qa.z, f.qa.w}, wb[4] = {f.qb.x, f.qb.y, f.qb.z, f.qb.w};
#pragma unroll
      for (int gi = 0; gi < kGroups; ++gi) {
        float c[kTiles][4];
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) c[j][e] = 0.f;
#pragma unroll
        for (int w = gi * 4 / kGroups; w < (gi + 1) * 4 / kGroups; ++w) {
          uint4 v[kTiles];
#pragma unroll
          for (int j = 0; j < kTiles; ++j)
            v[j] = *reinterpret_cast<const uint4*>(from + 8 * j * kMidRow + i * 256 + w * 64);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t a0, a1, a2, a3;
            decode_four<kHalf>(wa[w] >> (8 * half), a0, a2);
            decode_four<kHalf>(wb[w] >> (8 * half), a1, a3);
#pragma unroll
            for (int j = 0; j < kTiles; ++j)
              mma16816<kHalf>(c[j], a0, a1, a2, a3, half ? v[j].z : v[j].x, half ? v[j].w : v[j].y);
          }
        }
        const float s0 = scale_value(f.s[gi][0], kF32Scale, g & 1), s1 = scale_value(f.s[gi][1], kF32Scale, g & 1);
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
          if (on) {
            acc[j][0] += s0 * c[j][0];
            acc[j][1] += s0 * c[j][1];
            acc[j][2] += s1 * c[j][2];
            acc[j][3] += s1 * c[j][3];
          }
      }
    }
    __syncthreads();
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  // [token][row], a row more to a token's line against bank conflicts
  constexpr int kLine = kWarps * kRows + 1;
  static_assert(kTok * kLine * 4 <= mid_smem<kTiles>(), "the sums fit where the stages were");
  float* sums = reinterpret_cast<float*>(msm);
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      sums[(8 * j + 2 * t + (e & 1)) * kLine + warp * kRows + g + 8 * (e >> 1)] = acc[j][e];
  __syncthreads();
  if (splits > 1) cluster.sync();
  if (active) {
    // A thread has a row and every 2 splits-th token of it. Four of those at a
    // time: what another CTA holds is far away.
    static_assert(kWarps * 32 == 2 * kWarps * kRows, "two tokens at a time");
    const int r = threadIdx.x % (kWarps * kRows);
    const long long n = group_of * kWarps * kRows + r;
    const int step = 2 * splits;
    for (int m0 = 2 * blockIdx.x + threadIdx.x / (kWarps * kRows); m0 < kTok; m0 += 4 * step) {
      float v[4] = {};
      for (int k = 0; k < splits; ++k) {
        const float* from = splits > 1 ? cluster.map_shared_rank(sums, k) : sums;
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = from[min(m0 + i * step, kTok - 1) * kLine + r];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += w[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (m0 + i * step < M && n < N) y[(m0 + i * step) * ldy + n] = from_f<XT>(v[i]);
    }
  }
  if (splits > 1) cluster.sync();
}

// ---------------------------------------------------------------------- host

bool good_group(int g) { return g == 32 || g == 64 || g == 128; }

std::once_flag g_flags[kMaxDevices];
int g_ok[kMaxDevices];
int g_sms[kMaxDevices];

template <typename F>
int launch_cluster(F kernel, dim3 grid, int threads, int smem, int cluster, cudaStream_t s,
                   void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), args));
}

// CTAs of a cluster: as many (a power of two) as leave each warp a block and
// the GPU no more than about two CTAs an SM (a cluster's barriers cost more
// than a third CTA gains).
int pick_splits(long long tiles, long long steps, int sms) {
  int s = 1;
  while (s < kMaxCluster && tiles * s * 2 <= 2LL * sms + sms / 2 && steps >= (long long)s * 2 * kWarps) s *= 2;
  return s;
}

template <typename XT, typename ST, int kGroups>
int run_matvec(const void* x, long long ldx, const void* packed, const void* scales, int M, int N,
               int K, void* y, long long ldy, int sms, cudaStream_t s) {
  const int kblocks = (int)(((long long)K + kCols - 1) / kCols);
  const long long rtiles = ((long long)N + kRows - 1) / kRows;
  const int splits = pick_splits(rtiles, kblocks, sms);
  dim3 grid;
  if (!grid_of(rtiles, splits, &grid)) return TT_ERR_SHAPE;
  int wide = K % 8 == 0 && ldx % (16 / (int)sizeof(XT)) == 0 && aligned16(x);
  int kb = kblocks;
  void* args[] = {&x, &ldx, &packed, &scales, &M, &N, &K, &kb, &wide, &y, &ldy};
  return launch_cluster(matvec_kernel<XT, ST, kGroups>, grid, kWarps * 32, 0, splits, s, args);
}

template <typename XT, typename ST, int kTiles, int kGroups>
int run_mid(const void* x, long long ldx, const void* packed, const void* scales, int M, int N, int K, void* y,
            long long ldy, int sms, cudaStream_t s) {
  int kblocks = (int)(((long long)K + kCols - 1) / kCols);
  const long long groups = ((long long)N + kRows * kWarps - 1) / (kRows * kWarps);
  int splits = 1;  // two CTAs an SM, four blocks for each
  while (splits < kMaxCluster && groups * splits * 2 <= 2LL * sms && kblocks >= splits * 2 * kMidBlocks) splits *= 2;
  dim3 grid;
  if (!grid_of(groups, splits, &grid)) return TT_ERR_SHAPE;
  int wide = ldx % 8 == 0 && aligned16(x);
  void* args[] = {&x, &ldx, &packed, &scales, &M, &N, &K, &kblocks, &wide, &y, &ldy};
  return launch_cluster(mid_kernel<XT, ST, kTiles, kGroups>, grid, kWarps * 32, mid_smem<kTiles>(), splits, s, args);
}
template <typename XT, typename ST, int kTiles>
int run_mid_group(const void* x, long long ldx, const void* packed, const void* scales, int M, int N, int K, int group,
                  void* y, long long ldy, int sms, cudaStream_t s) {
  if (group == 128) return run_mid<XT, ST, kTiles, 1>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
  if (group == 64) return run_mid<XT, ST, kTiles, 2>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
  return run_mid<XT, ST, kTiles, 4>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
}

template <int kTiles>
constexpr int t_smem() { return kWarps * 8 * kTiles * (kCols + 4) * 4; }

template <typename XT, typename ST, int kTiles, int kGroups>
int run_matvec_t(const void* dy, long long lddy, const void* packed, const void* scales, int M,
                 int N, int K, void* dx, long long lddx, int sms, cudaStream_t s) {
  int kblocks = (int)(((long long)K + kCols - 1) / kCols);
  const long long rtiles = ((long long)N + kRows - 1) / kRows;
  const long long tiles = (long long)kblocks * (((long long)M + 8 * kTiles - 1) / (8 * kTiles));
  const int splits = pick_splits(tiles, rtiles, sms);
  dim3 grid;
  if (!grid_of(tiles, splits, &grid)) return TT_ERR_SHAPE;
  void* args[] = {&dy, &lddy, &packed, &scales, &M, &N, &K, &kblocks, &dx, &lddx};
  return launch_cluster(matvec_t_kernel<XT, ST, kTiles, kGroups>, grid, kWarps * 32, t_smem<kTiles>(), splits, s,
                        args);
}

template <typename F>
bool set_smem(F kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
}
template <typename XT, typename ST, int kGroups>
bool set_group() {
  bool ok = set_smem(matvec_t_kernel<XT, ST, 1, kGroups>, t_smem<1>());
  if constexpr (sizeof(XT) == 4) ok = ok && set_smem(matvec_t_kernel<XT, ST, 2, kGroups>, t_smem<2>());
  if constexpr (sizeof(XT) == 2)
    ok = ok && set_smem(mid_kernel<XT, ST, 2, kGroups>, mid_smem<2>()) &&
         set_smem(mid_kernel<XT, ST, 4, kGroups>, mid_smem<4>());
  return ok;
}
template <typename XT, typename ST>
int set_attrs() {
  return set_group<XT, ST, 1>() && set_group<XT, ST, 2>() && set_group<XT, ST, 4>() ? TT_OK : TT_ERR_CUDA;
}

int setup(int dev) {
  return once_per_device(g_flags, g_ok, dev, [dev]() -> int {
    if (cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return TT_ERR_CUDA;
    int st = set_attrs<float, float>();
    if (st == TT_OK) st = set_attrs<float, __nv_bfloat16>();
    if (st == TT_OK) st = set_attrs<__nv_bfloat16, float>();
    if (st == TT_OK) st = set_attrs<__nv_bfloat16, __nv_bfloat16>();
    if (st == TT_OK) st = set_attrs<__half, float>();
    if (st == TT_OK) st = set_attrs<__half, __nv_bfloat16>();
    return st;
  });
}

template <typename XT, typename ST>
int matmul_typed(bool transposed, const void* x, long long ldx, const void* packed,
                 const void* scales, int M, int N, int K, int group, void* y, long long ldy,
                 int sms, cudaStream_t s) {
  const int gpb = kCols / group;
  if (transposed) {
    if constexpr (sizeof(XT) == 4) {
      if (M > 8) {
        if (gpb == 1) return run_matvec_t<XT, ST, 2, 1>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
        if (gpb == 2) return run_matvec_t<XT, ST, 2, 2>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
        return run_matvec_t<XT, ST, 2, 4>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
      }
    }
    if (gpb == 1) return run_matvec_t<XT, ST, 1, 1>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
    if (gpb == 2) return run_matvec_t<XT, ST, 1, 2>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
    return run_matvec_t<XT, ST, 1, 4>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
  }
  if constexpr (sizeof(XT) == 2) {
    if (M > 16) return run_mid_group<XT, ST, 4>(x, ldx, packed, scales, M, N, K, group, y, ldy, sms, s);
    if (M > 8) return run_mid_group<XT, ST, 2>(x, ldx, packed, scales, M, N, K, group, y, ldy, sms, s);
  }
  if (gpb == 1) return run_matvec<XT, ST, 1>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
  if (gpb == 2) return run_matvec<XT, ST, 2>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
  return run_matvec<XT, ST, 4>(x, ldx, packed, scales, M, N, K, y, ldy, sms, s);
}

template <typename XT>
int matmul_scaled(bool transposed, const void* x, long long ldx, const void* packed,
                  const void* scales, int scale_type, int M, int N, int K, int group, void* y,
                  long long ldy, int sms, cudaStream_t s) {
  return scale_type == kF32
             ? matmul_typed<XT, float>(transposed, x, ldx, packed, scales, M, N, K, group, y, ldy, sms, s)
             : matmul_typed<XT, __nv_bfloat16>(transposed, x, ldx, packed, scales, M, N, K, group, y, ldy, sms, s);
}

int matmul(bool transposed, const void* x, int type, long long ldx, const void* packed,
           const void* scales, int scale_type, const float* row_scale, int M, int N, int K, int group,
           void* y, long long ldy, void* workspace, size_t workspace_bytes, int* dev_status, void* stream) {
  if (!x || !packed || !scales || !row_scale || !y || !dev_status) return TT_ERR_NULL;
  const bool few = M <= few_rows(type, transposed);
  if (!few && !workspace) return TT_ERR_NULL;
  if (M <= 0 || N <= 0 || K <= 0 || !good_group(group)) return TT_ERR_SHAPE;
  if (type < 0 || type > 2 || scale_type < 0 || scale_type > 1) return TT_ERR_SHAPE;
  if (ldx < (transposed ? N : K) || ldy < (transposed ? K : N)) return TT_ERR_SHAPE;
  if (!aligned16(packed) || !aligned16(scales)) return TT_ERR_ALIGN;
  int dev = 0;
  int st = check_device(&dev);
  if (st != TT_OK) return st;
  if ((st = setup(dev)) != TT_OK) return st;
  cudaStream_t s = (cudaStream_t)stream;
  const int sms = g_sms[dev];
  if (!few)
    return run_gemm(transposed, x, type, ldx, packed, scales, scale_type, row_scale, M, N, K, group, y, ldy,
                    workspace, workspace_bytes, dev_status, dev, s);
  if (type == kF32)
    return matmul_scaled<float>(transposed, x, ldx, packed, scales, scale_type, M, N, K, group, y, ldy, sms, s);
  if (type == kBF16)
    return matmul_scaled<__nv_bfloat16>(transposed, x, ldx, packed, scales, scale_type, M, N, K, group, y, ldy, sms, s);
  return matmul_scaled<__half>(transposed, x, ldx, packed, scales, scale_type, M, N, K, group, y, ldy, sms, s);
}

template <typename WT, typename ST>
int run_quantize(const void* W, long long ldw, int N, int K, int group, void* packed, void* scales,
                 cudaStream_t s) {
  const int kblocks = (int)(((long long)K + kCols - 1) / kCols);
  const long long blocks = ((long long)N + kRows - 1) / kRows * kblocks;
  const long long ctas = (blocks + 7) / 8;
  if (ctas > 0x7fffffffLL) return TT_ERR_SHAPE;
  quantize_kernel<WT, ST><<<(unsigned)ctas, 256, 0, s>>>((const WT*)W, ldw, N, K, group,
                                                         (uint4*)packed, (ST*)scales, blocks, kblocks);
  return cuda_status(cudaGetLastError());
}

template <typename OT, typename ST>
int run_dequantize(const void* packed, const void* scales, int N, int K, int group, void* out,
                   cudaStream_t s) {
  const int kblocks = (int)(((long long)K + kCols - 1) / kCols);
  const long long blocks = ((long long)N + kRows - 1) / kRows * kblocks;
  const long long ctas = (blocks + 7) / 8;
  if (ctas > 0x7fffffffLL) return TT_ERR_SHAPE;
  dequantize_kernel<OT, ST><<<(unsigned)ctas, 256, 0, s>>>((const uint4*)packed, (const ST*)scales, N, K,
                                                           group, (OT*)out, blocks, kblocks);
  return cuda_status(cudaGetLastError());
}

}  // namespace
}  // namespace q4
}  // namespace tt

extern "C" {

size_t tt_q4_packed_bytes(int N, int K) {
  if (N <= 0 || K <= 0) return 0;
  return ((size_t)N + 15) / 16 * (((size_t)K + 127) / 128) * tt::q4::kBlockBytes;
}

size_t tt_q4_scale_count(int N, int K, int group) {
  if (N <= 0 || K <= 0 || !tt::q4::good_group(group)) return 0;
  return ((size_t)N + 15) / 16 * (((size_t)K + 127) / 128) * (128 / group) * 16;
}

int tt_q4_pack(const signed char* codes, const void* scales, int scale_type, int N, int K, int group,
               void* packed, void* packed_scales, void* stream) {
  using namespace tt;
  if (!codes || !scales || !packed || !packed_scales) return TT_ERR_NULL;
  if (N <= 0 || K <= 0 || !q4::good_group(group) || scale_type < 0 || scale_type > 1) return TT_ERR_SHAPE;
  if (!aligned16(packed)) return TT_ERR_ALIGN;
  int st = check_device(nullptr);
  if (st != TT_OK) return st;
  const int kblocks = (int)(((long long)K + q4::kCols - 1) / q4::kCols);
  const long long blocks = ((long long)N + q4::kRows - 1) / q4::kRows * kblocks;
  const long long ctas = (blocks + 7) / 8;
  if (ctas > 0x7fffffffLL) return TT_ERR_SHAPE;
  cudaStream_t s = (cudaStream_t)stream;
  if (scale_type == q4::kF32)
    q4::pack_kernel<float><<<(unsigned)ctas, 256, 0, s>>>(codes, (const float*)scales, N, K, group,
                                                          (uint4*)packed, (float*)packed_scales, blocks, kblocks);
  else
    q4::pack_kernel<__nv_bfloat16><<<(unsigned)ctas, 256, 0, s>>>(
        codes, (const __nv_bfloat16*)scales, N, K, group, (uint4*)packed, (__nv_bfloat16*)packed_scales,
        blocks, kblocks);
  return cuda_status(cudaGetLastError());
}

int tt_q4_quantize(const void* W, int type, long long ldw, int scale_type, int N, int K, int group,
                   void* packed, void* packed_scales, void* stream) {
  using namespace tt;
  if (!W || !packed || !packed_scales) return TT_ERR_NULL;
  if (N <= 0 || K <= 0 || !q4::good_group(group) || ldw < K) return TT_ERR_SHAPE;
  if (type < 0 || type > 2 || scale_type < 0 || scale_type > 1) return TT_ERR_SHAPE;
  if (!aligned16(packed)) return TT_ERR_ALIGN;
  int st = check_device(nullptr);
  if (st != TT_OK) return st;
  cudaStream_t s = (cudaStream_t)stream;
  using BF = __nv_bfloat16;
  if (type == q4::kF32)
    return scale_type == q4::kF32 ? q4::run_quantize<float, float>(W, ldw, N, K, group, packed, packed_scales, s)
                                  : q4::run_quantize<float, BF>(W, ldw, N, K, group, packed, packed_scales, s);
  if (type == q4::kBF16)
    return scale_type == q4::kF32 ? q4::run_quantize<BF, float>(W, ldw, N, K, group, packed, packed_scales, s)
                                  : q4::run_quantize<BF, BF>(W, ldw, N, K, group, packed, packed_scales, s);
  return scale_type == q4::kF32 ? q4::run_quantize<__half, float>(W, ldw, N, K, group, packed, packed_scales, s)
                                : q4::run_quantize<__half, BF>(W, ldw, N, K, group, packed, packed_scales, s);
}

int tt_q4_dequantize(const void* packed, const void* packed_scales, int scale_type, int N, int K,
                     int group, void* out, int type, void* stream) {
  using namespace tt;
  if (!packed || !packed_scales || !out) return TT_ERR_NULL;
  if (N <= 0 || K <= 0 || !q4::good_group(group)) return TT_ERR_SHAPE;
  if (type < 0 || type > 2 || scale_type < 0 || scale_type > 1) return TT_ERR_SHAPE;
  if (!aligned16(packed)) return TT_ERR_ALIGN;
  int st = check_device(nullptr);
  if (st != TT_OK) return st;
  cudaStream_t s = (cudaStream_t)stream;
  using BF = __nv_bfloat16;
  if (type == q4::kF32)
    return scale_type == q4::kF32 ? q4::run_dequantize<float, float>(packed, packed_scales, N, K, group, out, s)
                                  : q4::run_dequantize<float, BF>(packed, packed_scales, N, K, group, out, s);
  if (type == q4::kBF16)
    return scale_type == q4::kF32 ? q4::run_dequantize<BF, float>(packed, packed_scales, N, K, group, out, s)
                                  : q4::run_dequantize<BF, BF>(packed, packed_scales, N, K, group, out, s);
  return scale_type == q4::kF32 ? q4::run_dequantize<__half, float>(packed, packed_scales, N, K, group, out, s)
                                : q4::run_dequantize<__half, BF>(packed, packed_scales, N, K, group, out, s);
}

int tt_q4_row_scale(const void* packed_scales, int scale_type, int N, int K, int group, float* row_scale,
                    void* stream) {
  using namespace tt;
  if (!packed_scales || !row_scale) return TT_ERR_NULL;
  if (N <= 0 || K <= 0 || !q4::good_group(group) || scale_type < 0 || scale_type > 1) return TT_ERR_SHAPE;
  int st = check_device(nullptr);
  if (st != TT_OK) return st;
  return q4::run_row_scale(packed_scales, scale_type, N, K, group, row_scale, (cudaStream_t)stream);
}

size_t tt_q4_matmul_workspace_bytes(int type, int scale_type, int transposed, int M, int N, int K) {
  if (type < 0 || type > 2 || N <= 0 || K <= 0 || M <= tt::q4::few_rows(type, transposed != 0)) return 0;
  return tt::q4::gemm_workspace_bytes(type, scale_type, transposed != 0, M, N, K);
}

int tt_q4_matmul(const void* x, int type, long long ldx, const void* packed, const void* packed_scales,
                 int scale_type, const float* row_scale, int M, int N, int K, int group, void* y, long long ldy,
                 void* workspace, size_t workspace_bytes, int* dev_status, void* stream) {
  return tt::q4::matmul(false, x, type, ldx, packed, packed_scales, scale_type, row_scale, M, N, K, group, y, ldy,
                        workspace, workspace_bytes, dev_status, stream);
}

int tt_q4_matmul_t(const void* dy, int type, long long lddy, const void* packed, const void* packed_scales,
                   int scale_type, const float* row_scale, int M, int N, int K, int group, void* dx,
                   long long lddx, void* workspace, size_t workspace_bytes, int* dev_status, void* stream) {
  return tt::q4::matmul(true, dy, type, lddy, packed, packed_scales, scale_type, row_scale, M, N, K, group, dx,
                        lddx, workspace, workspace_bytes, dev_status, stream);
}

}  // extern "C"
