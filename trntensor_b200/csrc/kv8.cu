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

constexpr int kThreads = 128;

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
};

// One CTA a page of a sequence, a head, and keys or values. The new tokens
// stand in shared memory as fp32 between the two passes (maximum, codes).
template <typename T>
__global__ void __launch_bounds__(kThreads) append_kernel(const Append p) {
  extern __shared__ float tile[];  // [token][dim]
  __shared__ unsigned int top;
  using q4::to_f;
  const int b = blockIdx.z;
  const int h = blockIdx.y >> 1, values = blockIdx.y & 1;
  const long long start = p.lengths[b];
  long long count = p.n_new ? p.n_new[b] : p.S;
  const bool first = blockIdx.y == 0;
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
    for (int o = 0; o < p.batch; ++o) {
      const long long so = p.lengths[o];
      const long long no = p.n_new ? p.n_new[o] : p.S;
      if (so < 0 || no <= 0) continue;
      const long long c1 = min((so + no - 1) / p.page, (long long)p.cols - 1);
      for (long long c = so / p.page + threadIdx.x; c <= c1; c += kThreads)
        if (!(o == b && c == col) && p.table[o * p.table_b + c] == page) raise(p.status, kSharedPage);
    }
  }
  const int slot0 = (int)(t0 - col * p.page), n = (int)(t1 - t0);
  const T* x = static_cast<const T*>(values ? p.v : p.k);
  const long long xs = values ? p.v_s : p.k_s;
  x += b * (values ? p.v_b : p.k_b) + (t0 - start) * xs + h * (values ? p.v_h : p.k_h);
  if (threadIdx.x == 0) top = 0;
  __syncthreads();
  unsigned int mine = 0;
  const int dim = p.dim;
  if (values || p.half == 0) {
    for (int i = threadIdx.x; i < n * dim; i += kThreads) {
      const float v = to_f(x[(long long)(i / dim) * xs + i % dim]);
      tile[i] = v;
      mine = max(mine, __float_as_uint(fabsf(v)));
    }
  } else {
    const int rest = dim - p.half;  // a thread a pair, or a lone value behind them
    for (int i = threadIdx.x; i < n * rest; i += kThreads) {
      const int tok = i / rest, j = i % rest;
      const T* row = x + tok * xs;
      float* out = tile + tok * dim;
      if (j < p.half) {
        const int a = p.interleaved ? 2 * j : j, c = p.interleaved ? 2 * j + 1 : j + p.half;
        float cs, sn;
        turn(t0 + tok, p.inv_freq[j], &cs, &sn);
        const float u = to_f(row[a]), w = to_f(row[c]);
        const float ru = u * cs - w * sn, rw = w * cs + u * sn;
        out[a] = ru;
        out[c] = rw;
        mine = max(mine, max(__float_as_uint(fabsf(ru)), __float_as_uint(fabsf(rw))));
      } else {
        const float v = to_f(row[j + p.half]);
        out[j + p.half] = v;
        mine = max(mine, __float_as_uint(fabsf(v)));
      }
    }
  }
  mine = __reduce_max_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) atomicMax(&top, mine);
  float* scale = (values ? p.vs : p.ks) + (long long)page * p.heads + h;
  const float old = slot0 == 0 ? 0.f : *scale;
  __syncthreads();
  const float nan = __int_as_float(0x7fffffff);
  const float need = top >= 0x7f800000u ? nan : __fdiv_rn(__uint_as_float(top), 127.f);
  const float now = old != old || need != need ? nan : fmaxf(old, need);
  if (threadIdx.x == 0 && slot0 == 0) *scale = now;
  unsigned char* base = (values ? p.vc : p.kc) + ((long long)page * p.heads + h) * p.page * dim;
  if (slot0 > 0 && now > old) {  // earlier tokens onto the larger scale
    const float ratio = __fdiv_rn(old, now);
    if (values) {
      for (int i = threadIdx.x; i < (slot0 + 15) / 16 * dim; i += kThreads) {
        const int unit = i / dim, have = min(16, slot0 - unit * 16);
        unsigned char* at = base + (long long)i * 16;
        for (int e = 0; e < have; ++e)
          at[e] = (unsigned char)((int)rintf((float)((int)at[e] - 128) * ratio) + 128);
      }
    } else {
      for (int i = threadIdx.x; i < slot0 * dim; i += kThreads)
        base[i] = (unsigned char)((int)rintf((float)((int)base[i] - 128) * ratio) + 128);
    }
  }
  if (slot0 > 0) {
    __syncthreads();  // every thread has read the old scale
    if (threadIdx.x == 0) *scale = now;
  }
  for (int i = threadIdx.x; i < n * dim; i += kThreads) {
    const int tok = i / dim, d = i % dim, slot = slot0 + tok;
    const float c = now > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(tile[i], now)), -127.f), 127.f) : 0.f;
    const unsigned char q = (unsigned char)((int)c + 128);
    if (values)
      base[(long long)(slot / 16) * 16 * dim + d * 16 + slot % 16] = q;
    else
      base[(long long)slot * dim + d] = q;
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

// Pages as values: k, v (n, heads, page, dim), each s c rounded once. A page
// id outside the cache reads as zeros.
template <typename T>
__global__ void __launch_bounds__(kThreads)
read_kernel(const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc,
            const float* __restrict__ ks, const float* __restrict__ vs, const int* __restrict__ ids,
            T* __restrict__ k, T* __restrict__ v, int* status, int pages, int heads, int page, int dim) {
  using q4::from_f;
  const int h = blockIdx.y;
  const long long id = ids ? ids[blockIdx.x] : blockIdx.x;
  const long long to = ((long long)blockIdx.x * heads + h) * page * dim;
  if (id < 0 || id >= pages) {
    if (threadIdx.x == 0 && h == 0) raise(status, kBadPage);
    for (int i = threadIdx.x; i < page * dim; i += kThreads) k[to + i] = v[to + i] = from_f<T>(0.f);
    return;
  }
  const long long from = (id * heads + h) * page * dim;
  const float sk = ks[id * heads + h], sv = vs[id * heads + h];
  for (int i = threadIdx.x; i < page * dim / 16; i += kThreads) {
    const uint4 q = *reinterpret_cast<const uint4*>(kc + from + 16LL * i);
    const unsigned char* c = reinterpret_cast<const unsigned char*>(&q);
#pragma unroll
    for (int e = 0; e < 16; ++e) k[to + 16LL * i + e] = from_f<T>(sk * (float)((int)c[e] - 128));
  }
  for (int i = threadIdx.x; i < page * dim / 16; i += kThreads) {
    const uint4 q = *reinterpret_cast<const uint4*>(vc + from + 16LL * i);
    const unsigned char* c = reinterpret_cast<const unsigned char*>(&q);
    const int unit = i / dim, d = i % dim;
#pragma unroll
    for (int e = 0; e < 16; ++e)
      v[to + (long long)(unit * 16 + e) * dim + d] = from_f<T>(sv * (float)((int)c[e] - 128));
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
    const int bytes = 128 * 256 * 4;
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
  const dim3 grid(most, 2u * heads, batch);
  const int smem = (S < page ? S : page) * dim * 4;
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
  if (!aligned16(k_codes) || !aligned16(v_codes)) return TT_ERR_ALIGN;
  int st = check_device(nullptr);
  if (st != TT_OK) return st;
  const dim3 grid(count, heads);
  cudaStream_t s = (cudaStream_t)stream;
  const unsigned char *kc = (const unsigned char*)k_codes, *vc = (const unsigned char*)v_codes;
  if (type == q4::kF32)
    kv8::read_kernel<float><<<grid, kv8::kThreads, 0, s>>>(kc, vc, k_scales, v_scales, page_ids, (float*)k,
                                                           (float*)v, status, pages, heads, page, dim);
  else if (type == q4::kBF16)
    kv8::read_kernel<__nv_bfloat16><<<grid, kv8::kThreads, 0, s>>>(
        kc, vc, k_scales, v_scales, page_ids, (__nv_bfloat16*)k, (__nv_bfloat16*)v, status, pages, heads, page, dim);
  else
    kv8::read_kernel<__half><<<grid, kv8::kThreads, 0, s>>>(kc, vc, k_scales, v_scales, page_ids, (__half*)k,
                                                            (__half*)v, status, pages, heads, page, dim);
  return cuda_status(cudaGetLastError());
}

}  // extern "C"
