// Attention of few query rows over a paged 8-bit cache (csrc/kv8.cuh).
//
//   o = sum_t softmax_t(scale q.K^[t]) V^[t],  K^[t] = sk[page,h] ck[t]
//
// Two contractions with a softmax between; the scores stay in registers. A
// kv head's query rows (tokens x heads of its group) make tiles of 8 or 16, and
// the work is cut into chunks of 64 tokens of one tile. The chunks of all
// sequences, heads and tiles form one line, of which every warp takes an equal
// piece, so that ragged lengths and a lone long sequence both fill the GPU. A
// tile whose chunks lie with several warps is joined in shared memory when
// they are of one CTA, and by a second small kernel when they are not, always
// in the same order.
//
// What bounds it: the cache's bytes, and close behind them the instructions
// that decode and multiply (with rows on the 16-wide side of the fragments,
// half of it empty, they took a third more time). bf16, 128 a head: 64
// sequences of 4400 to 8192 tokens x 8 kv heads 149 us (5.5 TB/s of cache), one of
// 131000 tokens 57 us (4.7 TB/s); three of 100 tokens 13 us, launches and waits.
// Each warp keeps its own ring of shared memory slots (one unit quartet of keys or
// of values each) filled by bulk copies two or three slots ahead, across tile
// borders. Tensor-core operands: the codes are exact in fp16; a row of q is scaled by a power of two
// to below 2^14 and rounded to fp16 (exact for 16-bit types down to 2^-27 of the
// row's largest value, 2^-39 of that below) or, for fp32, kept as two fp16
// terms. The softmax weights are fp16 (2^-11 of each, an eighth of a bf16
// result's rounding and as much as an fp16 one's; again held up by 2^14), two
// terms for fp32. Page scales enter in fp32: keys' into the exponent, and
// values' too, so that a weight times its value scale is what a row's maximum is
// of and what is rounded: scales of pages that a row does not see, or gives no
// weight to, take no bits from the others.
//
// Fragments: tokens are the 16-wide side of both products, query rows the
// 8-wide one. Fragment s of a chunk has the tokens 4 s .. 4 s + 3 of its four
// units: its row 2 u + e is token 4 s + e of unit u, row 8 + 2 u + e token 4 s +
// 2 + e. So a lane's scores are all of one unit; eight by eight transposed
// (movmatrix) they are the second product's operand; and a lane reads sixteen
// neighbouring bytes of a key row, and all sixteen tokens of a value row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "kv8.cuh"
#include "ptx.cuh"
#include "q4.cuh"

namespace tt {
namespace kv8 {

constexpr int kChunk = 64;
// Chunks (a power of two) after which the sums of values of 16-bit types are put
// aside and start anew: the tensor cores cut off up to 2^-23 of them at every 16
// tokens, to one side, 1.1e-4 until then. (fp32 types empty theirs every chunk.)
constexpr int kLongRun = 256;
constexpr int kNever = 0x7fffff00;  // behind the last token that any row sees (lengths are at most this)
constexpr float kUp = 16384.f, kUpLog = 14.f;  // the largest fp16 weight of a chunk

struct Attend {
  const void* q;
  long long q_b, q_s, q_h;
  void* o;  // (batch, S, heads_q, dim) contiguous
  const unsigned char* kc;
  const unsigned char* vc;
  const float* ks;
  const float* vs;
  const int* table;
  long long table_b;
  const int* lengths;
  const int* n_query;  // nullable: S
  float* part;         // pieces: [CTA][warp][2][16][2 + dim] (maximum, sum, values)
  float* joint;        // and joined: [CTA][2][16][2 + dim]
  int4* meta;          // [CTA]: (b, h * tiles + tile, last CTA, 1) of a tile that others finish
  int* places;         // prefill_kernel, above `most` tokens: [SM] 1 where the place is taken, zeros at first
  float* aside;        // and the places: [SM][dim][256 rows]
  int* status;
  float scale;  // times log2(e)
  int causal;
  int batch, S, heads_q, heads, dim, page, page_log, pages, cols, rows, tiles, tile_rows, sms, most;
};

template <int DP>
struct Shape {
  // Measured for 32 x 1 over 8192 with 8 kv heads (us): 128 wide 8 x 2 83, 8 x 3
  // 86, 12 x 2 110; 192 wide 6 x 2 124, 4 x 2 141, 4 x 3 133; 256 wide 4 x 3 170,
  // 4 x 2 189, 6 x 2 190.
  static constexpr int kWarps = DP <= 128 ? 8 : DP == 192 ? 6 : 4;
  static constexpr int kUnit = 16 * DP;
  static constexpr int kSlot = 4 * (kUnit + 32) + 32;  // four units; with keys their scales, and the values'
  static constexpr int kSlots = DP == 256 ? 3 : 2;
  static constexpr int kSmem = kWarps * kSlots * kSlot;
  static_assert(kSmem + 1024 <= 227 * 1024, "shared memory of an SM");
};

// The key scale of a unit whose page is outside the cache: its tokens are hidden.
__device__ const float kGone = -1.f;

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
// Four bytes into shared memory (zeros where not `on`).
__device__ __forceinline__ void copy_scale(uint32_t dst, const float* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
// Notes on the barrier that all of this lane's earlier copies are there.
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float lds32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
// Bounded wait: false when the copy has not arrived within the budget.
__device__ __forceinline__ bool wait_full(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_drain(bar, parity);
}
// Sixteen neighbouring values, 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load16(const T* at, float (&x)[16]) {
  constexpr int kPer = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 16 / kPer; ++i) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(at) + i);
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[i * kPer + j] = q4::to_f(e[j]);
  }
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
// Four biased codes as two fp16 pairs.
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 ra = __hsub2(reinterpret_cast<const __half2&>(a), bias);
  const __half2 rb = __hsub2(reinterpret_cast<const __half2&>(b), bias);
  lo = reinterpret_cast<const uint32_t&>(ra);
  hi = reinterpret_cast<const uint32_t&>(rb);
}
// A value scale as 2^lg x odd, with lg in -80 .. 125, and back = 2^-lg / up. lg
// goes into the exponent of the weights; odd is what is left: 1, or the scale's
// mantissa where lg is to be exact, and for a scale outside of the range (0,
// infinity, NaN and what is next to them) the rest of it. (Sums of weights reach
// 2^80 of the largest; the scale of a page of finite values is below 2^121. Scales
// in a row's sight may be 2^100 apart, or weights of the smaller ones are lost.)
struct Level {
  float lg, odd, back;
};
template <bool kExact>
__device__ __forceinline__ Level level_of(float s, float up) {
  Level v;
  const float c = fminf(fmaxf(s, 0x1p-80f), 0x1p125f);  // NaN: the least
  if constexpr (kExact) {
    const uint32_t e = __float_as_uint(c) >> 23;
    const float inv = __uint_as_float((254u - e) << 23);
    v.lg = (float)((int)e - 127);
    v.odd = s * inv;
    v.back = inv * (1.f / up);
  } else {
    const float inv = __fdividef(1.f, c);
    asm("lg2.approx.f32 %0, %1;" : "=f"(v.lg) : "f"(c));
    v.odd = s == c ? 1.f : s * inv;
    v.back = inv * (1.f / up);
  }
  return v;
}
// An 8 x 8 matrix of 16-bit values in fragment order, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Two floats (below 65504) as kTerms fp16 pairs.
template <int kTerms>
__device__ __forceinline__ void split_f16(float a, float b, uint32_t (&out)[kTerms]) {
#pragma unroll
  for (int i = 0; i < kTerms; ++i) {
    const __half2 v = __floats2half2_rn(a, b);
    out[i] = reinterpret_cast<const uint32_t&>(v);
    a -= __low2float(v);
    b -= __high2float(v);
  }
}

__device__ __forceinline__ long long clamp_length(const Attend& p, int b, bool report) {
  long long n = p.lengths[b];
  const long long most = (long long)p.cols * p.page;
  if (n < 0 || n > most) {
    if (report) raise(p.status, kBadLength);
    n = n < 0 ? 0 : most;
  }
  return n;
}
__device__ __forceinline__ int clamp_count(const Attend& p, int b, bool report) {
  int n = p.n_query ? p.n_query[b] : p.S;
  if (n < 0 || n > p.S) {
    if (report) raise(p.status, kBadLength);
    n = n < 0 ? 0 : p.S;
  }
  return n;
}
__device__ __forceinline__ long long chunks_of(long long n) { return (n + kChunk - 1) / kChunk; }

// Chunks of the sequences before `b_end`, summed by a warp.
__device__ __forceinline__ long long chunk_sum(const Attend& p, int b_end, int lane) {
  long long s = 0;
  for (int b = lane; b < b_end; b += 32) s += chunks_of(clamp_length(p, b, false));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s * p.heads * p.tiles;
}

// A place in the line of chunks.
struct Place {
  int b, h, tile;
  long long length;
  int chunk, chunks;
};

__device__ __forceinline__ void next_sequence(const Attend& p, Place& x) {
  x.h = x.tile = x.chunk = 0;
  do {
    ++x.b;
    x.length = x.b < p.batch ? clamp_length(p, x.b, false) : 0;
  } while (x.b < p.batch && x.length == 0);
  x.chunks = (int)chunks_of(x.length);
}
__device__ __forceinline__ void advance(const Attend& p, Place& x) {
  if (++x.chunk < x.chunks) return;
  x.chunk = 0;
  if (++x.tile < p.tiles) return;
  x.tile = 0;
  if (++x.h < p.heads) return;
  next_sequence(p, x);
}

// Pieces of a row (maximum, sum, values) made one by a warp: first the largest
// maximum, then the sums, so that the loads do not wait for one another.
template <int DP>
struct Joined {
  static constexpr int kPer = DP / 32;
  float m, l, a[kPer];
  // Pieces first, first + step, .. last, each `stride` floats behind the one
  // before; those that `there` marks as missing are left out. `head`: what
  // piece 0 lies behind its place.
  __device__ __forceinline__ void join(const float* in, int stride, int first, int last, int step, int dim, int lane,
                                       const int4* there, int head = 0) {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) a[e] = 0.f;
    for (int k = first + step * lane; k <= last; k += step * 32)
      if (there == nullptr || there[k].x >= 0) m = fmaxf(m, in[(long long)k * stride + (k == 0 ? head : 0)]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float z = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int k = first; k <= last; k += step) {
      if (there != nullptr && there[k].x < 0) continue;
      const float* at = in + (long long)k * stride + (k == 0 ? head : 0);
      const float f = exp2_approx(at[0] - z);
      l += at[1] * f;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (lane + 32 * e < dim) a[e] += at[2 + lane + 32 * e] * f;
    }
  }
  __device__ __forceinline__ void keep(float* out, int dim, int lane) const {
    if (lane == 0) {
      out[0] = m;
      out[1] = l;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (lane + 32 * e < dim) out[2 + lane + 32 * e] = a[e];
  }
  template <typename T>
  __device__ __forceinline__ void finish(T* o, int dim, int lane) const {
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (lane + 32 * e < dim) o[lane + 32 * e] = q4::from_f<T>(a[e] * inv);
  }
};
// Where row r of kv head h's rows stands in the result.
__device__ __forceinline__ long long row_offset(const Attend& p, int b, int h, int r) {
  const int group = p.heads_q / p.heads;
  return (((long long)b * p.S + r / group) * p.heads_q + h * group + r % group) * p.dim;
}

// NT: tiles of 8 rows that a warp has at a time. kLong: a warp may have more
// than kLongRun chunks of a tile.
template <typename T, int DP, int kTerms, int NT, bool kLong>
__global__ void __launch_bounds__(Shape<DP>::kWarps * 32, 1) attend_kernel(const Attend p) {
  using S = Shape<DP>;
  constexpr int kTile = 8 * NT;
  using q4::from_f;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t bars[S::kWarps * S::kSlots];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // pieces of tiles that this CTA's warps leave: tile, whether it began and ended here
  __shared__ int4 left_at[S::kWarps * 2];
  if (threadIdx.x < S::kWarps * 2) left_at[threadIdx.x] = make_int4(-1, 0, 0, 0);
  // a copy of an earlier call never arrived, and nobody has looked at that yet:
  // what leaves here is NaN, as it is where a copy of this call does not arrive
  __shared__ int before;
  const int status = threadIdx.x == 0 ? *(volatile int*)p.status : 0;
  unsigned char* mine = smem + warp * S::kSlots * S::kSlot;
  uint64_t* bar = bars + warp * S::kSlots;
  const int dim = p.dim;
  const uint32_t unit_bytes = 16 * dim;

  if (lane < S::kSlots) mbar_init(bar + lane, 1 + 4);  // the units' bytes, and their scales
  fence_mbar_init();
  __syncwarp();

  // sequences without a token, and what is wrong with the lengths
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    const long long n = clamp_length(p, b, threadIdx.x == 0);
    if (threadIdx.x == 0) clamp_count(p, b, true);
    if (n == 0) {
      const long long all = (long long)p.S * p.heads_q * dim;
      for (long long i = threadIdx.x; i < all; i += blockDim.x)
        static_cast<T*>(p.o)[b * all + i] = from_f<T>(0.f);
    }
  }
  if (threadIdx.x == 0) {
    before = status & kTimeout;
    p.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // this warp's piece of the line
  const long long total = chunk_sum(p, p.batch, lane);
  // Warps of a CTA that work: one while there are no more chunks than CTAs, so
  // that a little work spreads over the SMs; each has a chunk at least.
  const int per_cta = (int)max(1LL, min((long long)S::kWarps, (total + gridDim.x - 1) / gridDim.x));
  const long long workers = min((long long)gridDim.x * per_cta, total);
  const long long worker = (long long)blockIdx.x * per_cta + warp;
  const bool works = warp < per_cta && worker < workers;
  const long long begin = works ? total * worker / workers : 0, end = works ? total * (worker + 1) / workers : 0;
  const int group = p.heads_q / p.heads;
  const int rows_of = dim + 2;
  if (works) {
  Place at;
  {
    // the last sequence that starts at or before `begin`
    long long before = 0;
    int found = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      const int b = b0 + lane;
      const long long c = b < p.batch ? chunks_of(clamp_length(p, b, false)) * p.heads * p.tiles : 0;
      long long sum = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const unsigned in = __ballot_sync(0xffffffffu, before + sum > begin);
      if (in) {
        const int first = __ffs(in) - 1;
        before += __shfl_sync(0xffffffffu, sum - c, first);
        found = b0 + first;
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    at.b = found;
    at.length = clamp_length(p, found, false);
    at.chunks = (int)chunks_of(at.length);
    const long long in = begin - before;
    at.chunk = (int)(in % at.chunks);
    at.tile = (int)(in / at.chunks % p.tiles);
    at.h = (int)(in / at.chunks / p.tiles);
  }

  // ---- copies: lane t (t < 4 of the warp) stands for unit t of a chunk
  Place ahead = at;              // the chunk whose keys are asked for next
  long long left = end - begin;  // chunks not yet asked for
  // page of this lane's unit of a place; -1 behind the sequence's end
  auto page_at = [&](const Place& x) -> int {
    const int tok = x.chunk * kChunk + 16 * t;
    if (tok >= (int)x.length) return -1;
    return p.table[x.b * p.table_b + (tok >> p.page_log)];
  };
  uint32_t slot_in = 0;
  // Keys bring both scales with them: the maxima are of scores with the values'.
  auto ask = [&](const unsigned char* codes, bool keys, bool gone, int page, int h, int tok) {
    const unsigned has = __ballot_sync(0xffffffffu, page >= 0) & 15u;
    uint64_t* b = bar + slot_in;
    unsigned char* to = mine + slot_in * S::kSlot;
    if (lane == 0) mbar_arrive_expect_tx(b, __popc(has) * unit_bytes);
    __syncwarp();
    if (lane < 4) {
      const long long head = (long long)max(page, 0) * p.heads + h;
      if (page >= 0)
        bulk_load(smem_u32(to + t * (S::kUnit + 32)),
                  codes + (head * p.page + (tok & (p.page - 1))) * dim, unit_bytes, smem_u32(b));
      if (keys) {
        copy_scale(smem_u32(to + 4 * (S::kUnit + 32) + 4 * t), gone ? &kGone : p.ks + head, gone || page >= 0);
        copy_scale(smem_u32(to + 4 * (S::kUnit + 32) + 16 + 4 * t), p.vs + head, page >= 0);
      }
      copies_arrive(smem_u32(b));
    }
    slot_in = slot_in + 1 == S::kSlots ? 0 : slot_in + 1;
  };

  // Copies are asked for in the order K0 V0 K1 V1 ..., always kSlots ahead.
  // page_k is the page of the chunk whose keys come next (read from the table
  // one chunk before it is used), the others are of the one whose keys were
  // asked for last.
  int page_k = page_at(ahead), page_v = -1, head_v = 0, tok_v = 0;
  bool want_values = false;  // the next copy is of values
  bool lost = false;         // a page outside the cache has come by: from there on, tokens are looked at one by one
  auto ask_next = [&]() {
    if (want_values) {
      ask(p.vc, false, false, page_v, head_v, tok_v);
      want_values = false;
      return;
    }
    if (left == 0) return;
    --left;
    const bool gone = page_k >= p.pages || (page_k < 0 && ahead.chunk * kChunk + 16 * t < (int)ahead.length);
    if (__any_sync(0xffffffffu, gone)) {
      lost = true;
      if (gone && g == 0) raise(p.status, kBadPage);
      if (gone) page_k = -1;
    }
    page_v = page_k;
    head_v = ahead.h;
    tok_v = ahead.chunk * kChunk + 16 * t;
    ask(p.kc, true, gone, page_v, head_v, tok_v);
    want_values = true;
    if (left > 0) {
      advance(p, ahead);
      page_k = page_at(ahead);
    }
  };
  const long long stop = before == 0 ? end : begin;
  if (stop == end) {
#pragma unroll
    for (int i = 0; i < S::kSlots; ++i) ask_next();
  }

  uint32_t slot = 0, parity = 0;
  bool alive = true;
  auto arrive = [&]() {
    alive = __all_sync(0xffffffffu, wait_full(bar + slot, parity));
    if (!alive) {  // give up, but not before the other copies are in or the wait for them is over
      if (lane == 0) raise(p.status, kTimeout);
      for (uint32_t i = 0; i < S::kSlots; ++i) mbar_wait_drain(bar + i, i < slot ? parity ^ 1 : parity);
    }
  };
  auto release = [&]() {  // this slot's reads are done: the next copy goes into it
    fence_proxy_async_smem();
    __syncwarp();
    ask_next();
    slot = slot + 1 == S::kSlots ? 0 : slot + 1;
    if (slot == 0) parity ^= 1;
  };

  // Of rows 8 i + 2 t + e of the tile: maximum, sum, scale of the scores, tokens
  // that it sees. Sums of values: acc[i][n][e + 2 f] is d 16 n + 8 f + g.
  // Maxima are of a score in the exponent plus its unit's value scale there.
  float acc[NT][DP / 16][4], m[NT][2], l[NT][2], qs[NT][2];
  int lim[NT][2];
  uint32_t qf[NT][DP / 16][kTerms][2];
  int lim_min = 0;
  bool fresh = true, whole = true, aside = false;
  // The sums of values join those put aside before, in this warp's place for the
  // tile's piece: there, to start anew, or here, to leave (`back`).
  auto join_aside = [&](bool back) {
    float* base = p.part + (((long long)blockIdx.x * S::kWarps + warp) * 2 + (whole ? 1 : 0)) * 16 * rows_of;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float* out = base + (8 * a + 2 * t + e) * rows_of;
        const float top = m[a][e] == -INFINITY ? 0.f : m[a][e], keep = aside ? exp2_approx(out[0] - top) : 0.f;
        __syncwarp();
        if (g == 0) out[0] = m[a][e];
#pragma unroll
        for (int n = 0; n < DP / 16; ++n)
          if (16 * n < dim) {
            float x = acc[a][n][e], y = acc[a][n][e + 2];
            if (aside) {
              x += out[2 + 16 * n + g] * keep;
              y += out[2 + 16 * n + 8 + g] * keep;
            }
            if (!back) {
              out[2 + 16 * n + g] = x;
              out[2 + 16 * n + 8 + g] = y;
            }
            acc[a][n][e] = back ? x : 0.f;
            acc[a][n][e + 2] = back ? y : 0.f;
          }
      }
    __syncwarp();
    aside = !back;
  };

  long long i = begin;
  for (; i < stop; ++i) {
    if (fresh) {  // a tile begins: its queries
      fresh = false;
      whole = at.chunk == 0;
      const int count = clamp_count(p, at.b, false);
      lim_min = (int)at.length;
#pragma unroll
      for (int a = 0; a < NT; ++a) {
        // what rows 2 t, 2 t + 1 see; a row that is not there sees nothing
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = at.tile * kTile + 8 * a + 2 * t + e, tok = r / group;
          const bool has = r < p.rows && tok < count;
          const int see = !has ? 0 : max(p.causal ? (int)at.length - count + tok + 1 : (int)at.length, 0);
          lim[a][e] = see;
          if (has) lim_min = min(lim_min, see);
        }
        // the operand: row g
        const int r = at.tile * kTile + 8 * a + g, tok = r / group, head = at.h * group + r % group;
        const bool has = r < p.rows && tok < count;
        const T* row = static_cast<const T*>(p.q) + at.b * p.q_b + (has ? tok * p.q_s + head * p.q_h : 0);
        float x[DP / 64][16], top = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
          const int d = 16 * (t + 4 * c);
#pragma unroll
          for (int e = 0; e < 16; ++e) x[c][e] = 0.f;
          if (has && d < dim) load16(row + d, x[c]);
#pragma unroll
          for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[c][e]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // a row's power of two: its largest value comes to 2^13 .. 2^14
        int ex = (int)((__float_as_uint(top) >> 23) & 255);
        ex = ex < 14 ? 14 : ex;  // up = 2^(140 - ex), down = 1 / up
        const float up = __uint_as_float((uint32_t)(267 - ex) << 23) * (p.scale < 0.f ? -1.f : 1.f);
        const float down = __uint_as_float((uint32_t)(ex - 13) << 23) * fabsf(p.scale);
        qs[a][0] = __shfl_sync(0xffffffffu, down, 8 * t);
        qs[a][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float* y = x[c] + 4 * w;
            uint32_t lo[kTerms], hi[kTerms];
            split_f16<kTerms>(y[0] * up, y[1] * up, lo);
            split_f16<kTerms>(y[2] * up, y[3] * up, hi);
#pragma unroll
            for (int k = 0; k < kTerms; ++k) {
              qf[a][c * 4 + w][k][0] = lo[k];
              qf[a][c * 4 + w][k][1] = hi[k];
            }
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          m[a][e] = -INFINITY;
          l[a][e] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < DP / 16; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[a][n][e] = 0.f;
      }
      lim_min = __reduce_min_sync(0xffffffffu, lim_min);
    }

    // scores: sc[a][s][e + 2 f] is token 16 u + 4 s + 2 f + g % 2, u = g / 2, row 8 a + 2 t + e
    float sc[NT][4][4];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[a][j][e] = 0.f;
    arrive();
    if (!alive) break;
    {
      const uint32_t keys = smem_u32(mine + slot * S::kSlot) + (g >> 1) * (S::kUnit + 32) + (g & 1) * dim + t * 16;
#pragma unroll
      for (int c = 0; c < DP / 64; ++c)
#pragma unroll
        for (int j0 = 0; j0 < 4; j0 += 2) {
          uint4 va[2], vb[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            va[j] = lds128(keys + 4 * (j0 + j) * dim + c * 64);
            vb[j] = lds128(keys + (4 * (j0 + j) + 2) * dim + c * 64);
          }
          // fp32: an accumulator of these 64 d's own, as for the values below
          float own[kTerms == 2 ? NT : 1][2][4];
          if constexpr (kTerms == 2) {
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) own[a][j][e] = 0.f;
          }
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t a0, a1, a2, a3;
              decode4(w == 0 ? va[j].x : w == 1 ? va[j].y : w == 2 ? va[j].z : va[j].w, a0, a2);
              decode4(w == 0 ? vb[j].x : w == 1 ? vb[j].y : w == 2 ? vb[j].z : vb[j].w, a1, a3);
#pragma unroll
              for (int a = 0; a < NT; ++a)
#pragma unroll
                for (int k = 0; k < kTerms; ++k)
                  q4::mma16816<true>(kTerms == 2 ? own[a % (kTerms == 2 ? NT : 1)][j] : sc[a][j0 + j], a0, a1, a2, a3,
                                     qf[a][c * 4 + w][k][0], qf[a][c * 4 + w][k][1]);
            }
          if constexpr (kTerms == 2) {
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[a][j0 + j][e] += own[a][j][e];
          }
        }
    }
    float sk = lds32(smem_u32(mine + slot * S::kSlot) + 4 * (S::kUnit + 32) + 4 * (g >> 1));
    bool gone = false;
    if (lost) {
      gone = sk < 0.f;
      if (gone) sk = 0.f;
    }
    const Level sv = level_of<kTerms == 2>(lds32(smem_u32(mine + slot * S::kSlot) + 4 * (S::kUnit + 32) + 16 + 4 * (g >> 1)), kUp);
    release();

    // The scores are used as they are: scaled by f (at least 0, the same for a
    // lane's whole unit) only inside the exponent.
    int tok0 = at.chunk * kChunk + 16 * (g >> 1) + (g & 1);
    if (lost && gone) tok0 = kNever;
    const bool mask = (at.chunk + 1) * kChunk > lim_min || lost;
    if (mask) {
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (tok0 + 4 * j + (e & 2) >= lim[a][e & 1]) sc[a][j][e] = -INFINITY;
    }
    float f[NT][2], z[NT][2], old[NT][2];
    bool same = true;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        f[a][e] = qs[a][e] * sk;
        float n = fmaxf(sc[a][0][e], sc[a][0][e + 2]);
#pragma unroll
        for (int j = 1; j < 4; ++j) n = fmaxf(n, fmaxf(sc[a][j][e], sc[a][j][e + 2]));
        n = fmaxf(m[a][e], fmaf(n, f[a][e], sv.lg));  // what is not a number (a hidden unit of scale 0) drops out
        n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 4));
        n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 8));
        n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 16));
        z[a][e] = n == -INFINITY ? 0.f : n;
        old[a][e] = exp2_approx(m[a][e] - z[a][e]);
        m[a][e] = n;
        same = same && old[a][e] == 1.f;
      }
    if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
          acc[a][n][0] *= old[a][0];
          acc[a][n][1] *= old[a][1];
          acc[a][n][2] *= old[a][0];
          acc[a][n][3] *= old[a][1];
        }
    }
    // Weights times the unit's value scale, and times kUp. What is left of an odd
    // scale, or an exact one's mantissa, is multiplied after.
    uint32_t w[NT][4][kTerms][2];
    const bool plain = !mask && (kTerms == 2 || __all_sync(0xffffffffu, sv.odd == 1.f));
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      float sum[2] = {0.f, 0.f};
      const float y0 = (sv.lg + kUpLog) - z[a][0], y1 = (sv.lg + kUpLog) - z[a][1];
      if (plain) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sc[a][j][e] = exp2_approx(fmaf(sc[a][j][e], f[a][e & 1], e & 1 ? y1 : y0));
          sum[0] += sc[a][j][0] + sc[a][j][2];
          sum[1] += sc[a][j][1] + sc[a][j][3];
          if constexpr (kTerms == 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[a][j][e] *= sv.odd;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool hidden = mask && tok0 + 4 * j + (e & 2) >= lim[a][e & 1];
            const float v = hidden ? 0.f : exp2_approx(fmaf(sc[a][j][e], f[a][e & 1], e & 1 ? y1 : y0));
            sum[e & 1] += v;
            sc[a][j][e] = hidden ? 0.f : v * sv.odd;
          }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t lo[kTerms], hi[kTerms];
        split_f16<kTerms>(sc[a][j][0], sc[a][j][1], lo);
        split_f16<kTerms>(sc[a][j][2], sc[a][j][3], hi);
#pragma unroll
        for (int k = 0; k < kTerms; ++k) {
          w[a][j][k][0] = transpose8(lo[k]);
          w[a][j][k][1] = transpose8(hi[k]);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) l[a][e] = l[a][e] * old[a][e] + sum[e] * sv.back;
    }
    arrive();
    if (!alive) break;
    {
      const uint32_t vals = smem_u32(mine + slot * S::kSlot) + t * (S::kUnit + 32) + g * 16;
#pragma unroll
      for (int n0 = 0; n0 < DP / 16; n0 += 2) {
        uint4 va[2], vb[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          va[n] = lds128(vals + (n0 + n) * 256);
          vb[n] = lds128(vals + (n0 + n) * 256 + 128);
        }
        // fp32: an accumulator of the chunk's own, since the tensor cores cut
        // off at every addition (4e-6 of the result after 90 chunks)
        float own[kTerms == 2 ? NT : 1][2][4];
        if constexpr (kTerms == 2) {
#pragma unroll
          for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) own[a][n][e] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            uint32_t a0, a1, a2, a3;
            decode4(j == 0 ? va[n].x : j == 1 ? va[n].y : j == 2 ? va[n].z : va[n].w, a0, a2);
            decode4(j == 0 ? vb[n].x : j == 1 ? vb[n].y : j == 2 ? vb[n].z : vb[n].w, a1, a3);
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
              for (int k = 0; k < kTerms; ++k)
                q4::mma16816<true>(kTerms == 2 ? own[a % (kTerms == 2 ? NT : 1)][n] : acc[a][n0 + n], a0, a1, a2, a3,
                                   w[a][j][k][0], w[a][j][k][1]);
          }
        if constexpr (kTerms == 2) {
#pragma unroll
          for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[a][n0 + n][e] += own[a][n][e];
        }
      }
    }
    release();

    const bool last = at.chunk + 1 == at.chunks, leaves = last || i + 1 == end;
    if constexpr (kLong) {
      if (leaves ? aside : (at.chunk & (kLongRun - 1)) == kLongRun - 1) join_aside(leaves);
    }
    if (leaves) {  // the tile's sums leave the warp
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float den = l[a][e];
          den += __shfl_xor_sync(0xffffffffu, den, 4);
          den += __shfl_xor_sync(0xffffffffu, den, 8);
          den += __shfl_xor_sync(0xffffffffu, den, 16);
          const int in_tile = 8 * a + 2 * t + e, r = at.tile * kTile + in_tile;
          const bool none = lim[a][e] == 0;  // a row that sees nothing
          if (none) den = 0.f;
          if (r < p.rows) {
            if (whole && last) {
              const float inv = den > 0.f || den != den ? 1.f / (den * kUp) : 0.f;
              T* o = static_cast<T*>(p.o) + row_offset(p, at.b, at.h, r);
#pragma unroll
              for (int n = 0; n < DP / 16; ++n)
                if (16 * n < dim) {
                  o[16 * n + g] = from_f<T>(none ? 0.f : acc[a][n][e] * inv);
                  o[16 * n + 8 + g] = from_f<T>(none ? 0.f : acc[a][n][e + 2] * inv);
                }
            } else {
              // a piece for the joining: slot 0 of a tile that began before, 1 of one that goes on
              const float back_v = none ? 0.f : 1.f / kUp;
              float* out = p.part + (((long long)blockIdx.x * S::kWarps + warp) * 2 + (whole ? 1 : 0)) * 16 * rows_of +
                           in_tile * rows_of;
#pragma unroll
              for (int n = 0; n < DP / 16; ++n)
                if (16 * n < dim) {
                  out[2 + 16 * n + g] = none ? 0.f : acc[a][n][e] * back_v;
                  out[2 + 16 * n + 8 + g] = none ? 0.f : acc[a][n][e + 2] * back_v;
                }
              if (g == 0) *reinterpret_cast<float2*>(out) = make_float2(none ? -INFINITY : m[a][e], den);
            }
          }
        }
      if (!(whole && last) && lane == 0) {
        const long long c1 = i + (at.chunks - 1 - at.chunk);  // the tile's last chunk, and who has it
        const int who = (int)((((c1 + 1) * workers - 1) / total) / per_cta);
        left_at[warp * 2 + (whole ? 1 : 0)] =
            make_int4(at.b, at.h * p.tiles + at.tile, (whole ? 1 : 0) | (last ? 2 : 0), who);
      }
      fresh = true;
    }
    if (i + 1 < end) advance(p, at);
  }
  // What this warp has left to do is lost: NaN for each row that sees a token.
  for (; i < end; fresh = true) {
    if (fresh) whole = at.chunk == 0;
    const int rest = (int)min(end - i, (long long)(at.chunks - at.chunk)), count = clamp_count(p, at.b, false);
    const bool last = rest == at.chunks - at.chunk;
    for (int in_tile = 0; in_tile < kTile; ++in_tile) {
      const int r = at.tile * kTile + in_tile, tok = r / group;
      if (r >= p.rows) break;
      const bool none = tok >= count || (p.causal && (int)at.length - count + tok + 1 <= 0);
      const float lost = none ? 0.f : __int_as_float(0x7fffffff);
      if (whole && last) {
        T* o = static_cast<T*>(p.o) + row_offset(p, at.b, at.h, r);
        for (int d = lane; d < dim; d += 32) o[d] = from_f<T>(lost);
      } else {
        float* out = p.part + (((long long)blockIdx.x * S::kWarps + warp) * 2 + (whole ? 1 : 0)) * 16 * rows_of +
                     in_tile * rows_of;
        for (int d = lane; d < rows_of; d += 32) out[d] = d == 0 ? (none ? -INFINITY : 0.f) : lost;
      }
    }
    if (!(whole && last) && lane == 0) {
      const long long c1 = i + (at.chunks - 1 - at.chunk);
      left_at[warp * 2 + (whole ? 1 : 0)] = make_int4(at.b, at.h * p.tiles + at.tile, (whole ? 1 : 0) | (last ? 2 : 0),
                                                      (int)((((c1 + 1) * workers - 1) / total) / per_cta));
    }
    i += rest;
    at.chunk = at.chunks - 1;
    if (i < end) advance(p, at);
  }
  }  // works
  __syncthreads();
  // this CTA's pieces of a tile, one after the other in left_at, become one
  for (int i = 0; i < S::kWarps * 2;) {
    const int4 own = left_at[i];
    if (own.x < 0) {
      ++i;
      continue;
    }
    int j = i, flags = own.z;  // the first piece says whether it began here, the last whether it ended
    for (int k = i + 1; k < S::kWarps * 2; ++k) {
      const int4 o = left_at[k];
      if (o.x < 0) continue;
      if (o.x != own.x || o.y != own.y) break;
      j = k;
      flags |= o.z & 2;
    }
    const int h = own.y / p.tiles, tile = own.y % p.tiles;
    const bool begins = flags & 1, ends = flags & 2;
    for (int r = warp; r < kTile && tile * kTile + r < p.rows; r += S::kWarps) {
      const float* in = p.part + ((long long)blockIdx.x * S::kWarps * 2 * 16 + r) * rows_of;
      Joined<DP> x;
      x.join(in, 16 * rows_of, i, j, 1, dim, lane, left_at);
      if (begins && ends) {
        x.finish(static_cast<T*>(p.o) + row_offset(p, own.x, h, tile * kTile + r), dim, lane);
      } else {
        float* out = p.joint + (((long long)blockIdx.x * 2 + (begins ? 1 : 0)) * 16 + r) * rows_of;
        x.keep(out, dim, lane);
      }
    }
    if (begins && !ends && threadIdx.x == 0) p.meta[blockIdx.x] = make_int4(own.x, own.y, own.w, 1);
    i = j + 1;
  }
}

// Joins the pieces of the tiles that several CTAs had: one CTA for each that
// began such a tile, and each row of it; its warps share the pieces.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const Attend p) {
  constexpr int kW = 8;
  __shared__ float sums[kW][258];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early, runs after attend_kernel
  const int c0 = blockIdx.x;
  const int4 meta = p.meta[c0];
  const int row = meta.y % p.tiles * p.tile_rows + blockIdx.y, r = blockIdx.y;
  if (meta.w == 0 || row >= p.rows) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int rows_of = p.dim + 2;
  // slot 1 of the first CTA, slot 0 of those after it
  const float* in = p.joint + ((long long)c0 * 2 * 16 + r) * rows_of;
  Joined<256> x;
  x.join(in, 2 * 16 * rows_of, warp, meta.z - c0, kW, p.dim, lane, nullptr, 16 * rows_of);
  x.keep(sums[warp], p.dim, lane);
  __syncthreads();
  if (warp != 0) return;
  x.join(sums[0], 258, 0, kW - 1, 1, p.dim, lane, nullptr);
  x.finish(static_cast<T*>(p.o) + row_offset(p, meta.x, meta.y / p.tiles, row), p.dim, lane);
}

}  // namespace kv8
}  // namespace tt
