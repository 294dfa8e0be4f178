// Writing to and reading back a paged 8-bit key-value cache (csrc/kv8.cuh).
//
// Appending token t of sequence b: page = table[b][t / P], slot = t % P. For
// each page and head that a call touches
//   need = max |x| over the call's tokens in the page / 127,
//   s'   = max(s, need), where s counts as 0 when the call writes slot 0,
//   c    = rint(c s / s') for the earlier tokens where s' > s,
//   c    = rint(x / s') for the new ones;
// an infinity or NaN makes s' NaN. Keys are turned by their position first:
// (u, w) -> (u cos - w sin, w cos + u sin), angle t inv_freq[j], pairs
// (j, j + R/2) or (2 j, 2 j + 1).
// What bounds it: instructions (turning, maxima, rounding: 48 us of issue for
// the prompt below), then bytes. 8 kv heads of 128: a prompt of 2 x 8191 tokens in
// pages of 16, fp16, with its read back 60 us (2.8 TB/s), 64 sequences x 1 token
// in pages of 64, bf16, with theirs 16 us.
#include "common.cuh"
#include "kv8.cuh"
#include "q4.cuh"

namespace tt {
namespace kv8 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTableBytes = 128 * 128 * 8;  // cos and sin of a page's tokens, at most
// Page ids that a CTA's bits cover when it looks for pages written twice, and
// pages of a call (counted by its grid) up to which they are compared in pairs
// (one token for each of 64 sequences: 4.6 us, with bits 4.8; 272 pages 13.3 with
// either; 512 sequences 12.3 and 11.3; 32832 pages 4116 and 390).
constexpr int kBitsPages = 1 << 18;
constexpr int kPairs = 256;
static_assert(kBitsPages / 8 <= kWarps * 16 * 128 * 2, "the bits fit where the least staged tokens lie");

struct Append {
  const void* k;
  const void* v;
  long long k_b, k_s, k_h, v_b, v_s, v_h;  // strides in elements
  const int* table;
  long long table_b;
  const int* lengths;
  const int* n_new;  // nullable: S
  const float* inv_freq;
  int half, interleaved;
  unsigned char* kc;
  unsigned char* vc;
  float* ks;
  float* vs;
  int* status;
  int batch, S, heads, dim, page, pages, cols;
  int wide;  // rows can be read 16 bytes at a time
};

// Four codes rint(x / s) + 128 as bytes, as the division rounds them: x times
// the reciprocal is off by 127 2^-22 at most, so it decides unless it comes
// that near to a half; then, and for scales with no finite reciprocal, the
// division itself is made. |x| <= 127 s up to a rounding of s, so that codes need
// no clamping but where s is subnormal and that rounding large: a few units of
// 2^-149 for values of up to 190 such units. Adding 1.5 2^23 rounds to an
// integer, which then is the low byte.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float s, float inv, bool tiny) {
  constexpr float kRound = 12582912.f;
  uint32_t q[4];
  bool near = tiny;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float y = x[e] * inv, r = y + kRound;
    q[e] = __float_as_uint(r);
    near |= fabsf(y - (r - kRound)) > 0.49996f;
  }
  if (near) {
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
      const float y = __fdiv_rn(e == 0 ? x[0] : e == 1 ? x[1] : e == 2 ? x[2] : x[3], s);
      const uint32_t r = __float_as_uint(fminf(fmaxf(y, -127.f), 127.f) + kRound);
      if (e == 0) q[0] = r;
      else if (e == 1) q[1] = r;
      else if (e == 2) q[2] = r;
      else q[3] = r;
    }
  }
  return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410) ^ 0x80808080u;
}

// Four neighbouring values.
template <typename T>
__device__ __forceinline__ void four(const T* at, float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 f = *reinterpret_cast<const float4*>(at);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(at);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q4::to_f(e[i]);
  }
}

// A warp's new tokens of a page and head. kTurn: 0 as they stand, 1 turned in
// pairs (j, j + half), 2 in pairs (2 j, 2 j + 1). Sixteen tokens by 128 values
// at a time stand in the warp's part of shared memory (in registers they cost
// code for each of the sixteen, which the instruction caches did not hold).
constexpr int kRowTokens = 16, kRowValues = 128;
template <int kTurn, typename T>
struct Tokens {
  const T* x;           // the first
  long long stride;     // to the next
  const float2* cs;     // (cos, sin) by token and pair
  T* tile;              // [token][kRowValues]
  int n, half, dim;
  bool wide;            // 16-byte loads

  // Asks for tokens i0 .. at values d0 ..
  __device__ __forceinline__ void stage(int i0, int d0, int lane) const {
    constexpr int kPer = 16 / sizeof(T), kPieces = kRowValues / kPer;
    const int have = min(kRowTokens, n - i0) * kPieces;
#pragma unroll 4
    for (int i = lane; i < have; i += 32) {
      const int tok = i / kPieces, d = i % kPieces * kPer;
      if (d0 + d >= dim) continue;
      const T* from = x + (i0 + tok) * stride + d0 + d;
      T* to = tile + tok * kRowValues + d;
      if (wide) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
                     : "memory");
      } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) to[e] = from[e];
      }
    }
  }
  __device__ __forceinline__ void arrive() const {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
  }
  // Values d .. d + 3 of token i0 + i, of which the tile has those from d0 on.
  __device__ __forceinline__ void turned(int i0, int i, int d0, int d, float (&v)[4]) const {
    const T* at = tile + i * kRowValues + (d - d0);
    four(at, v);
    if (kTurn == 0 || d >= 2 * half) return;
    const float2* c = cs + (i0 + i) * half;
    if (kTurn == 2) {
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        if (d + e >= 2 * half) break;
        const float2 k = c[(d + e) / 2];
        const float u = v[e], w = v[e + 1];
        v[e] = u * k.x - w * k.y;
        v[e + 1] = w * k.x + u * k.y;
      }
    } else if (half % 4 == 0 && 2 * half <= kRowValues) {  // the four partners lie together, in the tile too
      const bool lead = d < half;
      float o[4];
      four(lead ? at + half : at - half, o);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 k = c[lead ? d + e : d + e - half];
        v[e] = lead ? v[e] * k.x - o[e] * k.y : v[e] * k.x + o[e] * k.y;
      }
    } else {
      const T* row = x + (i0 + i) * stride;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (d + e >= 2 * half) break;
        const bool lead = d + e < half;
        const float2 k = c[lead ? d + e : d + e - half];
        const float w = q4::to_f(row[lead ? d + e + half : d + e - half]);
        v[e] = lead ? v[e] * k.x - w * k.y : v[e] * k.x + w * k.y;
      }
    }
  }
};

// The new tokens' codes and their page's scale. kValues: values' storage order,
// else keys'. A lane has four neighbouring values of a token. The first tokens
// are asked for before the page is known (`ready` waits for the table), and a
// page's that all fit the tile are loaded once.
template <bool kValues, int kTurn, typename T, typename F>
__device__ __forceinline__ void put(const Append& p, const Tokens<kTurn, T>& in, int slot0, int h, int lane, F ready) {
  const int dim = p.dim, n = in.n;
  const bool once = n <= kRowTokens && dim <= kRowValues;
  in.stage(0, 0, lane);
  const int page = ready();
  if (page < 0) {
    in.arrive();
    return;
  }
  unsigned char* base = (kValues ? p.vc : p.kc) + ((long long)page * p.heads + h) * p.page * dim;
  float* scale = (kValues ? p.vs : p.ks) + (long long)page * p.heads + h;
  const float old = slot0 == 0 ? 0.f : *scale;
  in.arrive();
  uint32_t top = 0;  // largest magnitude by its bits, whose order puts infinities and NaN on top
  for (int i0 = 0; i0 < n; i0 += kRowTokens)
    for (int d0 = 0; d0 < dim; d0 += kRowValues) {
      if (i0 + d0 > 0) {
        __syncwarp();
        in.stage(i0, d0, lane);
        in.arrive();
      }
      const int d = d0 + 4 * lane;
      if (d < dim)
#pragma unroll 4
        for (int i = 0; i < min(kRowTokens, n - i0); ++i) {
          float v[4];
          in.turned(i0, i, d0, d, v);
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(fabsf(v[e])));
        }
    }
  top = __reduce_max_sync(0xffffffffu, top);
  const float nan = __int_as_float(0x7fffffff);
  const float need = top >= 0x7f800000u ? nan : __fdiv_rn(__uint_as_float(top), 127.f);
  const float now = old != old || need != need ? nan : fmaxf(old, need);
  __syncwarp();
  if (lane == 0) *scale = now;
  if (slot0 > 0 && now > old) {  // earlier tokens onto the larger scale
    const float ratio = __fdiv_rn(old, now);
    // keys: whole rows; values: a unit's 16 tokens of a d, of which the last unit keeps those behind slot0
    const int pieces = kValues ? (slot0 + 15) / 16 * dim : slot0 * dim / 16;
    for (int i = lane; i < pieces; i += 32) {
      uint4* at = reinterpret_cast<uint4*>(base) + i;
      const int have = kValues ? min(16, slot0 - i / dim * 16) : 16;
      uint4 q = *at;
      uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t c = (w[e / 4] >> (8 * (e % 4))) & 255u;
        const uint32_t r = (uint32_t)((int)rintf((float)((int)c - 128) * ratio) + 128);
        if (e < have) w[e / 4] ^= (c ^ r) << (8 * (e % 4));
      }
      *at = q;
    }
    __syncwarp();
  }
  const float inv = now > 0.f ? __fdiv_rn(1.f, now) : 0.f;
  const bool none = !(now > 0.f), tiny = now < 1e-36f;  // the reciprocal of a tiny scale is not finite
  for (int i0 = 0; i0 < n; i0 += kRowTokens)
    for (int d0 = 0; d0 < dim; d0 += kRowValues) {
      if (!once) {
        __syncwarp();
        in.stage(i0, d0, lane);
        in.arrive();
      }
      const int d = d0 + 4 * lane, have = min(kRowTokens, n - i0), slot = slot0 + i0;
      if (d >= dim) continue;
      if (!kValues || have < 16 || slot % 16 != 0) {
#pragma unroll 4
        for (int i = 0; i < have; ++i) {
          float v[4];
          in.turned(i0, i, d0, d, v);
          const uint32_t q = none ? 0x80808080u : codes_of(v, now, inv, tiny);
          if constexpr (!kValues) {
            *reinterpret_cast<uint32_t*>(base + (long long)(slot + i) * dim + d) = q;
          } else {
            unsigned char* at = base + ((long long)((slot + i) / 16) * dim + d) * 16 + (slot + i) % 16;
#pragma unroll
            for (int e = 0; e < 4; ++e) at[16 * e] = (unsigned char)(q >> (8 * e));
          }
        }
      } else {  // a whole unit of values
        uint32_t w[4][4];  // [d][four tokens]
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t row[4];  // four codes of a token
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float v[4];
            in.turned(i0, 4 * j + i, d0, d, v);
            row[i] = none ? 0x80808080u : codes_of(v, now, inv, tiny);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e][j] = __byte_perm(__byte_perm(row[0], row[1], 0x0040 + 0x11 * e),
                                  __byte_perm(row[2], row[3], 0x0040 + 0x11 * e), 0x5410);
        }
        uint4* at = reinterpret_cast<uint4*>(base + ((long long)(slot / 16) * dim + d) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) at[e] = make_uint4(w[e][0], w[e][1], w[e][2], w[e][3]);
      }
    }
}

// Pages that the call writes for two places, where there are too many to compare
// each with each: a bit for each page id of a part of them, which finds its
// second setting. A thread asks for four pages of the call's grid at a time.
__device__ __forceinline__ void find_shared(const Append& p, uint32_t* bits, int part) {
  const int first = part * kBitsPages, ids = min(kBitsPages, p.pages - first), shift = 31 - __clz(p.page);
  for (int i = threadIdx.x; i < (ids + 31) / 32; i += kThreads) bits[i] = 0;
  __syncthreads();
  const unsigned most = gridDim.x, step_b = kThreads / most, step_c = kThreads % most;
  unsigned b = threadIdx.x / most, c = threadIdx.x % most;  // the sequence, and the column behind its first
  bool twice = false;
  while (b < (unsigned)p.batch) {
    int start[4], count[4], id[4];
    unsigned at_b[4], at_c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      at_b[i] = b;
      at_c[i] = c;
      const bool in = b < (unsigned)p.batch;
      start[i] = in ? p.lengths[b] : -1;
      count[i] = in && p.n_new ? p.n_new[b] : p.S;
      b += step_b;
      c += step_c;
      if (c >= most) {
        c -= most;
        ++b;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long col = ((long long)start[i] >> shift) + at_c[i], end = (long long)start[i] + min(count[i], p.S);
      // a sequence that adds nothing writes no page
      const bool in = start[i] >= 0 && count[i] > 0 && col << shift < end && col < p.cols;
      id[i] = in ? p.table[at_b[i] * p.table_b + col] : -1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (id[i] < first || id[i] - first >= ids) continue;
      const uint32_t at = id[i] - first, bit = 1u << (at & 31);
      twice |= (atomicOr(bits + at / 32, bit) & bit) != 0;
    }
  }
  if (twice) raise(p.status, kSharedPage);
  __syncthreads();
}

// A warp takes a page of a sequence, a head, and keys or values. The CTA's
// warps are neighbouring heads, which share the table of cosines; the CTAs of
// the last y look for pages that the call writes for two places: each compares
// its own with all others or, where they are many (kMany), the first few go over
// all with bits in shared memory.
// Bound by bytes: k and v read once from HBM, codes written once.
template <typename T, bool kMany>
__global__ void __launch_bounds__(kThreads, 4) append_kernel(const Append p) {
  extern __shared__ __align__(16) unsigned char append_smem[];
  float2* table = reinterpret_cast<float2*>(append_smem + kWarps * kRowTokens * kRowValues * sizeof(T));  // [token][pair]
  const int b = blockIdx.z, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const bool look = blockIdx.y + 1 == gridDim.y;
  const long long all = (long long)p.batch * gridDim.x;
  if (kMany && look)
    for (long long part = (long long)blockIdx.z * gridDim.x + blockIdx.x; part * kBitsPages < p.pages; part += all)
      find_shared(p, reinterpret_cast<uint32_t*>(append_smem), (int)part);
  const long long start = p.lengths[b];
  long long count = p.n_new ? p.n_new[b] : p.S;
  if (start < 0 || count < 0 || count > p.S || start + count > (long long)p.cols * p.page) {
    if (look && blockIdx.x == 0 && threadIdx.x == 0) raise(p.status, kBadLength);
    if (start < 0) return;
    count = count < 0 ? 0 : count > p.S ? p.S : count;
  }
  const long long col = start / p.page + blockIdx.x;
  const long long t0 = max(start, col * p.page), t1 = min(start + count, (col + 1) * p.page);
  if (t0 >= t1 || col >= p.cols) return;
  const int page = p.table[b * p.table_b + col];
  if (look) {
    if (page < 0 || page >= p.pages) {
      if (threadIdx.x == 0) raise(p.status, kBadPage);
      return;
    }
    for (long long i = threadIdx.x; !kMany && i < all; i += kThreads) {
      const int o = (int)(i / gridDim.x);
      const long long so = p.lengths[o], no = min((long long)(p.n_new ? p.n_new[o] : p.S), (long long)p.S);
      const long long c = so / p.page + i % gridDim.x;
      // a sequence that adds nothing writes no page
      if (so >= 0 && no > 0 && c * p.page < so + no && c < p.cols && !(o == b && c == col) &&
          p.table[o * p.table_b + c] == page)
        raise(p.status, kSharedPage);
    }
    return;
  }
  const int slot0 = (int)(t0 - col * p.page), n = (int)(t1 - t0);
  const bool turns = blockIdx.y * kWarps < p.heads && p.half > 0;  // keys are among this CTA's
  const int task = blockIdx.y * kWarps + warp;
  const bool values = task >= p.heads;
  const int h = min(values ? task - p.heads : task, p.heads - 1);  // behind the last: for the barrier alone
  T* tile = reinterpret_cast<T*>(append_smem) + warp * kRowTokens * kRowValues;
  // between a warp's loads and their use: the table of cosines, and the page
  auto ready = [&]() -> int {
    if (turns) {
      for (int i = threadIdx.x; i < n * p.half; i += kThreads) {
        float c, sn;
        turn(t0 + i / p.half, p.inv_freq[i % p.half], &c, &sn);
        table[i] = make_float2(c, sn);
      }
      __syncthreads();
    }
    return task >= 2 * p.heads || page < 0 || page >= p.pages ? -1 : page;
  };
  if (values) {
    const T* x = static_cast<const T*>(p.v) + b * p.v_b + (t0 - start) * p.v_s + h * p.v_h;
    put<true, 0, T>(p, {x, p.v_s, table, tile, n, p.half, p.dim, p.wide != 0}, slot0, h, lane, ready);
  } else {
    const T* x = static_cast<const T*>(p.k) + b * p.k_b + (t0 - start) * p.k_s + h * p.k_h;
    if (p.half == 0)
      put<false, 0, T>(p, {x, p.k_s, table, tile, n, p.half, p.dim, p.wide != 0}, slot0, h, lane, ready);
    else if (!p.interleaved)
      put<false, 1, T>(p, {x, p.k_s, table, tile, n, p.half, p.dim, p.wide != 0}, slot0, h, lane, ready);
    else
      put<false, 2, T>(p, {x, p.k_s, table, tile, n, p.half, p.dim, p.wide != 0}, slot0, h, lane, ready);
  }
}

// x (batch, S, heads, dim) turned to the positions lengths[b] + i.
template <typename T>
__global__ void rotate_kernel(const T* __restrict__ x, long long x_b, long long x_s, long long x_h,
                              const int* __restrict__ lengths, const float* __restrict__ inv_freq,
                              int half, int interleaved, T* __restrict__ out, int S, int heads, int dim) {
  using q4::from_f;
  using q4::to_f;
  const int s = blockIdx.x, b = blockIdx.y;
  const long long t = (long long)lengths[b] + s;
  const T* row = x + b * x_b + s * x_s;
  T* to = out + ((long long)b * S + s) * heads * dim;
  extern __shared__ float cs[];  // cos, sin of each frequency
  for (int j = threadIdx.x; j < half; j += blockDim.x) turn(t, inv_freq[j], cs + 2 * j, cs + 2 * j + 1);
  __syncthreads();
  const int rest = dim - half;
  for (int i = threadIdx.x; i < heads * rest; i += blockDim.x) {
    const int h = i / rest, j = i % rest;
    const T* r = row + h * x_h;
    T* o = to + (long long)h * dim;
    if (j < half) {
      const int a = interleaved ? 2 * j : j, c = interleaved ? 2 * j + 1 : j + half;
      const float u = to_f(r[a]), w = to_f(r[c]);
      o[a] = from_f<T>(u * cs[2 * j] - w * cs[2 * j + 1]);
      o[c] = from_f<T>(w * cs[2 * j] + u * cs[2 * j + 1]);
    } else {
      o[j + half] = r[j + half];
    }
  }
}

// Sixteen values in as few stores as their type takes.
template <typename T, int N>
__device__ __forceinline__ void store_values(T* at, const float (&v)[N]) {
  constexpr int kWords = N * sizeof(T) / 4;
  uint32_t w[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
    else if constexpr (std::is_same<T, __half>::value) w[i] = q4::pack_f16(v[2 * i], v[2 * i + 1]);
    else w[i] = q4::pack_bf16(v[2 * i], v[2 * i + 1]);
  }
  if constexpr (kWords == 2) {
    *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kWords; i += 4)
      reinterpret_cast<uint4*>(at)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
}

// Pages as values: k, v (n, heads, page, dim), each s c rounded once. A page
// id outside the cache reads as zeros. One warp a page, head and half (keys or
// values).
template <typename T>
__global__ void __launch_bounds__(kThreads)
read_kernel(const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc,
            const float* __restrict__ ks, const float* __restrict__ vs, const int* __restrict__ ids,
            T* __restrict__ k, T* __restrict__ v, int* status, int count, int pages, int heads, int page, int dim) {
  using q4::from_f;
  const int lane = threadIdx.x & 31;
  const long long task = (long long)blockIdx.x * kWarps + threadIdx.x / 32;
  if (task >= (long long)count * heads * 2) return;
  const bool values = task & 1;
  const int h = (int)((task >> 1) % heads);
  const long long i0 = (task >> 1) / heads;
  const long long id = ids ? ids[i0] : i0;
  T* to = (values ? v : k) + (i0 * heads + h) * page * dim;
  if (id < 0 || id >= pages) {
    if (lane == 0 && h == 0) raise(status, kBadPage);
    for (int i = lane; i < page * dim; i += 32) to[i] = from_f<T>(0.f);
    return;
  }
  const unsigned char* from = (values ? vc : kc) + (id * heads + h) * page * dim;
  const float s = (values ? vs : ks)[id * heads + h];
  if (!values) {
#pragma unroll 2
    for (int i = lane; i < page * dim / 8; i += 32) {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(from) + i);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = s * (float)((int)((e < 4 ? q.x >> (8 * e) : q.y >> (8 * (e - 4))) & 255u) - 128);
      store_values<T, 8>(to + 8LL * i, x);
    }
  } else {
    for (int i = lane; i < page / 16 * dim / 4; i += 32) {  // four d of a unit's 16 tokens
      const int unit = i / (dim / 4), d = i % (dim / 4) * 4;
      uint32_t w[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(from) + (long long)unit * dim + d + j);
        w[j][0] = q.x; w[j][1] = q.y; w[j][2] = q.z; w[j][3] = q.w;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = s * (float)((int)((w[j][e / 4] >> (8 * (e % 4))) & 255u) - 128);
        store_values<T, 4>(to + (long long)(unit * 16 + e) * dim + d, x);
      }
    }
  }
}

bool good_shape(int pages, int heads, int page, int dim) {
  return pages > 0 && heads > 0 && heads <= 32767 &&
         (page == 16 || page == 32 || page == 64 || page == 128) && dim >= 16 && dim <= 256 && dim % 16 == 0;
}

template <typename T>
bool set_append(int bytes) {
  const auto at = cudaFuncAttributeMaxDynamicSharedMemorySize;
  return cudaFuncSetAttribute(append_kernel<T, false>, at, bytes) == cudaSuccess &&
         cudaFuncSetAttribute(append_kernel<T, true>, at, bytes) == cudaSuccess;
}
template <typename T>
int run_append(const Append& p, dim3 grid, int smem, cudaStream_t s) {
  if ((long long)p.batch * grid.x > kPairs) append_kernel<T, true><<<grid, kThreads, smem, s>>>(p);
  else append_kernel<T, false><<<grid, kThreads, smem, s>>>(p);
  return cuda_status(cudaGetLastError());
}

std::once_flag g_flags[kMaxDevices];
int g_ok[kMaxDevices];

int setup(int dev) {
  return once_per_device(g_flags, g_ok, dev, []() -> int {
    const int bytes = kTableBytes + kWarps * kRowTokens * kRowValues * 4;
    if (!set_append<float>(bytes) || !set_append<__nv_bfloat16>(bytes) || !set_append<__half>(bytes))
      return TT_ERR_CUDA;
    return TT_OK;
  });
}

}  // namespace
}  // namespace kv8
}  // namespace tt

extern "C" {

int tt_kv8_append(const void* k, const void* v, int type, long long k_stride_b, long long k_stride_s,
                  long long k_stride_h, long long v_stride_b, long long v_stride_s,
                  long long v_stride_h, const int* block_table, long long table_stride, int columns,
                  const int* lengths, const int* n_new, const float* inv_freq, int pairs,
                  int interleaved, void* k_codes, void* v_codes, float* k_scales, float* v_scales,
                  int* status, int batch, int S, int heads, int dim, int page, int pages,
                  void* stream) {
  using namespace tt;
  if (!k || !v || !block_table || !lengths || !k_codes || !v_codes || !k_scales || !v_scales || !status)
    return TT_ERR_NULL;
  if (pairs > 0 && !inv_freq) return TT_ERR_NULL;
  if (batch <= 0 || batch > 65535 || S <= 0 || columns <= 0 || type < 0 || type > 2) return TT_ERR_SHAPE;
  if (!kv8::good_shape(pages, heads, page, dim) || pairs < 0 || 2 * pairs > dim) return TT_ERR_SHAPE;
  if (!aligned16(k_codes) || !aligned16(v_codes)) return TT_ERR_ALIGN;
  int dev = 0;
  int st = check_device(&dev);
  if (st != TT_OK) return st;
  if ((st = kv8::setup(dev)) != TT_OK) return st;
  kv8::Append p;
  p.k = k; p.v = v;
  p.k_b = k_stride_b; p.k_s = k_stride_s; p.k_h = k_stride_h;
  p.v_b = v_stride_b; p.v_s = v_stride_s; p.v_h = v_stride_h;
  p.table = block_table; p.table_b = table_stride; p.lengths = lengths; p.n_new = n_new;
  p.inv_freq = inv_freq; p.half = pairs; p.interleaved = interleaved;
  p.kc = (unsigned char*)k_codes; p.vc = (unsigned char*)v_codes;
  p.ks = k_scales; p.vs = v_scales; p.status = status;
  p.batch = batch; p.S = S; p.heads = heads; p.dim = dim; p.page = page; p.pages = pages; p.cols = columns;
  // S tokens lie in at most this many pages, wherever they start
  const unsigned most = (unsigned)(((long long)S + page - 2) / page + 1);
  const dim3 grid(most, (2u * heads + kv8::kWarps - 1) / kv8::kWarps + 1, batch);
  const int size = type == q4::kF32 ? 4 : 2;
  const int smem = (S < page ? S : page) * pairs * 8 + kv8::kWarps * kv8::kRowTokens * kv8::kRowValues * size;
  const int per = 16 / size;
  p.wide = aligned16(k) && aligned16(v) && k_stride_b % per == 0 && k_stride_s % per == 0 && k_stride_h % per == 0 &&
           v_stride_b % per == 0 && v_stride_s % per == 0 && v_stride_h % per == 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (type == q4::kF32) return kv8::run_append<float>(p, grid, smem, s);
  if (type == q4::kBF16) return kv8::run_append<__nv_bfloat16>(p, grid, smem, s);
  return kv8::run_append<__half>(p, grid, smem, s);
}

int tt_kv8_rotate(const void* x, int type, long long stride_b, long long stride_s, long long stride_h,
                  const int* lengths, const float* inv_freq, int pairs, int interleaved, void* out,
                  int batch, int S, int heads, int dim, void* stream) {
  using namespace tt;
  if (!x || !lengths || !inv_freq || !out) return TT_ERR_NULL;
  if (batch <= 0 || batch > 65535 || S <= 0 || heads <= 0 || dim <= 0 || dim > 4096) return TT_ERR_SHAPE;
  if (pairs <= 0 || 2 * pairs > dim || type < 0 || type > 2) return TT_ERR_SHAPE;
  int st = check_device(nullptr);
  if (st != TT_OK) return st;
  const dim3 grid(S, batch);
  const int smem = pairs * 8;
  cudaStream_t s = (cudaStream_t)stream;
  if (type == q4::kF32)
    kv8::rotate_kernel<float><<<grid, 256, smem, s>>>((const float*)x, stride_b, stride_s, stride_h, lengths,
                                                      inv_freq, pairs, interleaved, (float*)out, S, heads, dim);
  else if (type == q4::kBF16)
    kv8::rotate_kernel<__nv_bfloat16><<<grid, 256, smem, s>>>(
        (const __nv_bfloat16*)x, stride_b, stride_s, stride_h, lengths, inv_freq, pairs, interleaved,
        (__nv_bfloat16*)out, S, heads, dim);
  else
    kv8::rotate_kernel<__half><<<grid, 256, smem, s>>>((const __half*)x, stride_b, stride_s, stride_h, lengths,
                                                       inv_freq, pairs, interleaved, (__half*)out, S, heads, dim);
  return cuda_status(cudaGetLastError());
}

int tt_kv8_read(const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales,
                const int* page_ids, int count, void* k, void* v, int type, int* status, int pages,
                int heads, int page, int dim, void* stream) {
  using namespace tt;
  if (!k_codes || !v_codes || !k_scales || !v_scales || !k || !v || !status) return TT_ERR_NULL;
  if (count <= 0 || (!page_ids && count > pages) || type < 0 || type > 2) return TT_ERR_SHAPE;
  if (!kv8::good_shape(pages, heads, page, dim)) return TT_ERR_SHAPE;
  if (!aligned16(k_codes) || !aligned16(v_codes) || !aligned16(k) || !aligned16(v)) return TT_ERR_ALIGN;
  int st = check_device(nullptr);
  if (st != TT_OK) return st;
  const long long ctas = ((long long)count * heads * 2 + kv8::kWarps - 1) / kv8::kWarps;
  if (ctas > 0x7fffffffLL) return TT_ERR_SHAPE;
  const unsigned grid = (unsigned)ctas;
  cudaStream_t s = (cudaStream_t)stream;
  const unsigned char *kc = (const unsigned char*)k_codes, *vc = (const unsigned char*)v_codes;
  if (type == q4::kF32)
    kv8::read_kernel<float><<<grid, kv8::kThreads, 0, s>>>(kc, vc, k_scales, v_scales, page_ids, (float*)k,
                                                           (float*)v, status, count, pages, heads, page, dim);
  else if (type == q4::kBF16)
    kv8::read_kernel<__nv_bfloat16><<<grid, kv8::kThreads, 0, s>>>(
        kc, vc, k_scales, v_scales, page_ids, (__nv_bfloat16*)k, (__nv_bfloat16*)v, status, count, pages, heads, page, dim);
  else
    kv8::read_kernel<__half><<<grid, kv8::kThreads, 0, s>>>(kc, vc, k_scales, v_scales, page_ids, (__half*)k,
                                                            (__half*)v, status, count, pages, heads, page, dim);
  return cuda_status(cudaGetLastError());
}

}  // extern "C"
