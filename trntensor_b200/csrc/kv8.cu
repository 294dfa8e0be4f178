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
#include "common.cuh"
#include "kv8.cuh"
#include "q4.cuh"

namespace tt {
namespace kv8 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTableBytes = 128 * 128 * 8;  // cos and sin of a page's tokens, at most

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
  int wide;  // four neighbouring values can be read at once
};

template <typename T>
__device__ __forceinline__ void load4(const T* at, bool wide, float (&v)[4]) {
  if (wide) {
    if constexpr (sizeof(T) == 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(at));
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(at));
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = q4::to_f(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q4::to_f(__ldg(at + i));
  }
}

// Values d .. d + 3 of a token, turned: kTurn 0 as they stand, 1 pairs (j, j +
// half), 2 pairs (2 j, 2 j + 1). cs: the token's (cos, sin) by pair.
template <int kTurn, typename T>
__device__ __forceinline__ void load_turned(const Append& p, const T* row, int d, const float2* cs, float (&v)[4]) {
  load4(row + d, p.wide, v);
  if (kTurn == 0 || d >= 2 * p.half) return;
  if (kTurn == 2) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      if (d + i >= 2 * p.half) break;
      const float2 a = cs[(d + i) / 2];
      const float u = v[i], w = v[i + 1];
      v[i] = u * a.x - w * a.y;
      v[i + 1] = w * a.x + u * a.y;
    }
  } else if (p.half % 4 == 0) {  // the four partners lie together
    const bool lead = d < p.half;
    float o[4];
    load4(row + (lead ? d + p.half : d - p.half), p.wide, o);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = cs[lead ? d + i : d + i - p.half];
      v[i] = lead ? v[i] * a.x - o[i] * a.y : v[i] * a.x + o[i] * a.y;
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      if (d + i >= 2 * p.half) break;
      const bool lead = d + i < p.half;
      const float2 a = cs[lead ? d + i : d + i - p.half];
      const float w = q4::to_f(row[lead ? d + i + p.half : d + i - p.half]), u = q4::to_f(row[d + i]);
      const float r = lead ? u * a.x - w * a.y : u * a.x + w * a.y;
      if (i == 0) v[0] = r;
      else if (i == 1) v[1] = r;
      else if (i == 2) v[2] = r;
      else v[3] = r;
    }
  }
}

// Four codes rint(x / s) + 128 as bytes, as the division rounds them: x times
// the reciprocal is off by 127 2^-22 at most, so it decides unless it comes
// that near to a half; then, and for scales with no finite reciprocal, the
// division itself is made.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float s, float inv, bool tiny) {
  float q[4];
  bool near = tiny;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float y = x[e] * inv;
    q[e] = rintf(y);
    near |= fabsf(y - q[e]) > 0.49996f;
  }
  if (near) {
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
      const float r = rintf(__fdiv_rn(e == 0 ? x[0] : e == 1 ? x[1] : e == 2 ? x[2] : x[3], s));
      if (e == 0) q[0] = r;
      else if (e == 1) q[1] = r;
      else if (e == 2) q[2] = r;
      else q[3] = r;
    }
  }
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) w |= (uint32_t)((int)fminf(fmaxf(q[e], -127.f), 127.f) + 128) << (8 * e);
  return w;
}

// Largest magnitude, by its bits, of a warp's tokens; and their codes.
template <int kTurn, typename T>
__device__ __forceinline__ uint32_t top_of(const Append& p, const T* x, long long xs, int n, const float2* cs, int lane) {
  uint32_t top = 0;
  for (int d = 4 * lane; d < p.dim; d += 128)
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      float v[4];
      load_turned<kTurn>(p, x + i * xs, d, cs + i * p.half, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(fabsf(v[e])));
    }
  return __reduce_max_sync(0xffffffffu, top);
}
template <int kTurn, typename T>
__device__ __forceinline__ void put_keys(const Append& p, const T* x, long long xs, int n, const float2* cs, int lane,
                                         unsigned char* to, float s, float inv, bool none, bool tiny) {
  for (int d = 4 * lane; d < p.dim; d += 128)
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      float v[4];
      load_turned<kTurn>(p, x + i * xs, d, cs + i * p.half, v);
      *reinterpret_cast<uint32_t*>(to + (long long)i * p.dim + d) = none ? 0x80808080u : codes_of(v, s, inv, tiny);
    }
}

// A warp takes a page of a sequence, a head, and keys or values: once over the
// new tokens for their largest value, once for the codes (from L1 or L2). The
// CTA's warps are neighbouring heads, which share the table of cosines.
// Bound by bytes: k and v read once from HBM, codes written once.
template <typename T>
__global__ void __launch_bounds__(kThreads) append_kernel(const Append p) {
  extern __shared__ float2 table[];  // [token][pair]
  const int b = blockIdx.z, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const bool first = blockIdx.y == 0;
  const long long start = p.lengths[b];
  long long count = p.n_new ? p.n_new[b] : p.S;
  if (start < 0 || count < 0 || count > p.S || start + count > (long long)p.cols * p.page) {
    if (first && blockIdx.x == 0 && threadIdx.x == 0) raise(p.status, kBadLength);
    if (start < 0) return;
    count = count < 0 ? 0 : count > p.S ? p.S : count;
  }
  const long long col = start / p.page + blockIdx.x;
  const long long t0 = max(start, col * p.page), t1 = min(start + count, (col + 1) * p.page);
  if (t0 >= t1 || col >= p.cols) return;
  const int page = p.table[b * p.table_b + col];
  if (page < 0 || page >= p.pages) {
    if (first && threadIdx.x == 0) raise(p.status, kBadPage);
    return;
  }
  if (first) {  // is the page written for another place too?
    const long long all = (long long)p.batch * gridDim.x;
    for (long long i = threadIdx.x; i < all; i += kThreads) {
      const int o = (int)(i / gridDim.x);
      const long long so = p.lengths[o], no = min((long long)(p.n_new ? p.n_new[o] : p.S), (long long)p.S);
      const long long c = so / p.page + i % gridDim.x;
      if (so >= 0 && c * p.page < so + no && c < p.cols && !(o == b && c == col) &&
          p.table[o * p.table_b + c] == page)
        raise(p.status, kSharedPage);
    }
  }
  const int slot0 = (int)(t0 - col * p.page), n = (int)(t1 - t0), dim = p.dim;
  const bool keys_here = blockIdx.y * kWarps < p.heads;
  if (keys_here && p.half > 0) {
    for (int i = threadIdx.x; i < n * p.half; i += kThreads) {
      float c, sn;
      turn(t0 + i / p.half, p.inv_freq[i % p.half], &c, &sn);
      table[i] = make_float2(c, sn);
    }
    __syncthreads();
  }
  const int task = blockIdx.y * kWarps + warp;
  if (task >= 2 * p.heads) return;
  const bool values = task >= p.heads;
  const int h = values ? task - p.heads : task;
  const T* x = static_cast<const T*>(values ? p.v : p.k);
  const long long xs = values ? p.v_s : p.k_s;
  x += b * (values ? p.v_b : p.k_b) + (t0 - start) * xs + h * (values ? p.v_h : p.k_h);
  const int mode = values || p.half == 0 ? 0 : p.interleaved ? 2 : 1;
  const uint32_t top = mode == 0 ? top_of<0>(p, x, xs, n, table, lane)
                       : mode == 1 ? top_of<1>(p, x, xs, n, table, lane) : top_of<2>(p, x, xs, n, table, lane);
  float* scale = (values ? p.vs : p.ks) + (long long)page * p.heads + h;
  const float nan = __int_as_float(0x7fffffff);
  const float old = slot0 == 0 ? 0.f : *scale;
  const float need = top >= 0x7f800000u ? nan : __fdiv_rn(__uint_as_float(top), 127.f);
  const float now = old != old || need != need ? nan : fmaxf(old, need);
  __syncwarp();
  if (lane == 0) *scale = now;
  unsigned char* base = (values ? p.vc : p.kc) + ((long long)page * p.heads + h) * p.page * dim;
  if (slot0 > 0 && now > old) {  // earlier tokens onto the larger scale
    const float ratio = __fdiv_rn(old, now);
    // keys: whole rows; values: a unit's 16 tokens of a d, of which the last unit keeps those behind slot0
    const int pieces = values ? (slot0 + 15) / 16 * dim : slot0 * dim / 16;
    for (int i = lane; i < pieces; i += 32) {
      uint4* at = reinterpret_cast<uint4*>(base) + i;
      const int have = values ? min(16, slot0 - i / dim * 16) : 16;
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
  if (!values) {
    unsigned char* to = base + (long long)slot0 * dim;
    if (mode == 0) put_keys<0>(p, x, xs, n, table, lane, to, now, inv, none, tiny);
    else if (mode == 1) put_keys<1>(p, x, xs, n, table, lane, to, now, inv, none, tiny);
    else put_keys<2>(p, x, xs, n, table, lane, to, now, inv, none, tiny);
    return;
  }
  for (int unit = slot0 / 16; unit * 16 < slot0 + n; ++unit) {
    const int lo = max(slot0 - unit * 16, 0), hi = min(slot0 + n - unit * 16, 16);
    for (int d = 4 * lane; d < dim; d += 128) {
      uint32_t row[16];  // four codes of a token
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        row[i] = 0x80808080u;
        if (i >= lo && i < hi && !none) {
          float v[4];
          load4(x + (unit * 16 + i - slot0) * xs + d, p.wide, v);
          row[i] = codes_of(v, now, inv, tiny);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        unsigned char* at = base + ((long long)unit * dim + d + e) * 16;
        if (hi - lo == 16) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a = __byte_perm(row[4 * j], row[4 * j + 1], 0x0040 + 0x11 * e);
            const uint32_t c = __byte_perm(row[4 * j + 2], row[4 * j + 3], 0x0040 + 0x11 * e);
            w[j] = __byte_perm(a, c, 0x5410);
          }
          *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i >= lo && i < hi) at[i] = (unsigned char)(row[i] >> (8 * e));
        }
      }
    }
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

std::once_flag g_flags[kMaxDevices];
int g_ok[kMaxDevices];

int setup(int dev) {
  return once_per_device(g_flags, g_ok, dev, []() -> int {
    const int bytes = kTableBytes;
    const auto at = cudaFuncAttributeMaxDynamicSharedMemorySize;
    if (cudaFuncSetAttribute(append_kernel<float>, at, bytes) != cudaSuccess ||
        cudaFuncSetAttribute(append_kernel<__nv_bfloat16>, at, bytes) != cudaSuccess ||
        cudaFuncSetAttribute(append_kernel<__half>, at, bytes) != cudaSuccess)
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
  const dim3 grid(most, (2u * heads + kv8::kWarps - 1) / kv8::kWarps, batch);
  const int smem = (S < page ? S : page) * pairs * 8;
  const int size = type == q4::kF32 ? 4 : 2;
  p.wide = ((uintptr_t)k | (uintptr_t)v) % (4 * size) == 0 && k_stride_b % 4 == 0 && k_stride_s % 4 == 0 &&
           k_stride_h % 4 == 0 && v_stride_b % 4 == 0 && v_stride_s % 4 == 0 && v_stride_h % 4 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (type == q4::kF32) kv8::append_kernel<float><<<grid, kv8::kThreads, smem, s>>>(p);
  else if (type == q4::kBF16) kv8::append_kernel<__nv_bfloat16><<<grid, kv8::kThreads, smem, s>>>(p);
  else kv8::append_kernel<__half><<<grid, kv8::kThreads, smem, s>>>(p);
  return cuda_status(cudaGetLastError());
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
