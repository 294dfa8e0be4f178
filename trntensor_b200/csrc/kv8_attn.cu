// Attention over a paged 8-bit cache: launches (csrc/kv8_attn.cuh).
#include "common.cuh"
#include "kv8_attn.cuh"
#include "kv8_prefill.cuh"

namespace tt {
namespace kv8 {
namespace {

std::once_flag g_flags[kMaxDevices];
int g_ok[kMaxDevices];
int g_sms[kMaxDevices];

template <typename T, int DP, int NT>
int set_attr() {
  constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;
  const auto at = cudaFuncAttributeMaxDynamicSharedMemorySize;
  if (cudaFuncSetAttribute(attend_kernel<T, DP, kTerms, NT, false>, at, Shape<DP>::kSmem) != cudaSuccess) return TT_ERR_CUDA;
  if constexpr (kTerms == 1)
    if (cudaFuncSetAttribute(attend_kernel<T, DP, kTerms, NT, true>, at, Shape<DP>::kSmem) != cudaSuccess) return TT_ERR_CUDA;
  return TT_OK;
}
template <typename T, int DP>
int set_prefill() {
  const auto at = cudaFuncAttributeMaxDynamicSharedMemorySize;
  return cudaFuncSetAttribute(prefill_kernel<T, DP, true, false>, at, PreShape<DP>::kSmem) == cudaSuccess &&
                 cudaFuncSetAttribute(prefill_kernel<T, DP, false, false>, at, PreShape<DP>::kSmem) == cudaSuccess &&
                 cudaFuncSetAttribute(prefill_kernel<T, DP, true, true>, at, PreShape<DP>::kSmem) == cudaSuccess &&
                 cudaFuncSetAttribute(prefill_kernel<T, DP, false, true>, at, PreShape<DP>::kSmem) == cudaSuccess
             ? TT_OK
             : TT_ERR_CUDA;
}
template <typename T>
int set_attrs() {
  int st = set_attr<T, 64, 1>();
  if (st == TT_OK) st = set_attr<T, 64, 2>();
  if (st == TT_OK) st = set_attr<T, 128, 1>();
  if (st == TT_OK) st = set_attr<T, 128, 2>();
  if (st == TT_OK) st = set_attr<T, 192, 1>();
  if (st == TT_OK) st = set_attr<T, 256, 1>();
  if constexpr (sizeof(T) == 2) {
    if (st == TT_OK) st = set_prefill<T, 64>();
    if (st == TT_OK) st = set_prefill<T, 128>();
  }
  return st;
}

int setup(int dev) {
  return once_per_device(g_flags, g_ok, dev, [dev]() -> int {
    if (cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return TT_ERR_CUDA;
    int st = set_attrs<float>();
    if (st == TT_OK) st = set_attrs<__nv_bfloat16>();
    if (st == TT_OK) st = set_attrs<__half>();
    return st;
  });
}

// One CTA an SM; for each a word of meta, two pieces a warp, and two joined.
int warps_of(int dim) { return dim <= 128 ? Shape<128>::kWarps : dim <= 192 ? Shape<192>::kWarps : Shape<256>::kWarps; }
size_t piece_bytes(int dim) { return (size_t)2 * 16 * (dim + 2) * 4; }
size_t workspace_bytes(int dim, int sms) { return sms * (16 + (warps_of(dim) + 1) * piece_bytes(dim)); }

template <typename T, int DP, int NT>
void launch_rows(const Attend& p, int sms, cudaStream_t s) {
  constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;
  using S = Shape<DP>;
  // What long runs need is left out where no warp can have one, even if all
  // sequences fill the table: it costs registers (32 x 16 rows over 8192 tokens, 128
  // a head, 128 against 135 us, 8 rows over 131000 58 against 61).
  const long long chunks = ((long long)p.cols * p.page + kChunk - 1) / kChunk;
  const long long share = chunks * p.tiles * p.heads * p.batch / (sms * S::kWarps) + 1;
  if constexpr (kTerms == 1) {
    if (chunks > kLongRun && share > kLongRun) {
      attend_kernel<T, DP, kTerms, NT, true><<<sms, S::kWarps * 32, S::kSmem, s>>>(p);
      return;
    }
  }
  attend_kernel<T, DP, kTerms, NT, false><<<sms, S::kWarps * 32, S::kSmem, s>>>(p);
}
template <typename T, int DP>
int launch(Attend p, int sms, cudaStream_t s) {
  // More than eight rows go sixteen at a time, which decodes the cache once for
  // both halves, where the registers hold them.
  p.tile_rows = p.rows <= 8 || DP > 128 ? 8 : 16;
  p.tiles = (p.rows + p.tile_rows - 1) / p.tile_rows;
  if (p.tile_rows == 8) {
    launch_rows<T, DP, 1>(p, sms, s);
  } else {
    if constexpr (DP <= 128) launch_rows<T, DP, 2>(p, sms, s);
  }
  int st = cuda_status(cudaGetLastError());
  if (st != TT_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms, p.rows < p.tile_rows ? p.rows : p.tile_rows);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, join_kernel<T>, p));
}
// 16-bit types with up to 128 values a head go to the tensor cores' tiles of
// 256 rows where that is faster. There 64 tokens take about 2850 clocks of a
// CTA (2250 if no more than 128 rows are used), however few of the SMs have
// one, and the other kernel about 620 of an SM for each 16 rows, spread over
// all SMs: the first wins from rows x heads x sequences = 64 (48) an SM for each
// wave of CTAs. (8192 tokens, 128 a head: 16 x 8 x 40 rows 153 against 149 us,
// 16 x 8 x 80 rows 152 against 238, 1 x 8 x 400 rows 190 against 110.)
bool many_rows(const Attend& p, int sms) {
  const long long tiles = ((long long)p.rows + 255) / 256 * p.heads * p.batch, waves = (tiles + sms - 1) / sms;
  return p.rows > 16 && (long long)p.rows * p.heads * p.batch > (p.rows > 128 ? 64 : 48) * waves * sms;
}

template <typename T, int DP, bool kLong>
int launch_tiles(const Attend& p, cudaStream_t s) {
  const long long tiles = ((long long)p.rows + 255) / 256;
  const dim3 grid((unsigned)tiles, p.heads, p.batch);
  if (p.dim == DP) prefill_kernel<T, DP, true, kLong><<<grid, kPreThreads, PreShape<DP>::kSmem, s>>>(p);
  else prefill_kernel<T, DP, false, kLong><<<grid, kPreThreads, PreShape<DP>::kSmem, s>>>(p);
  return cuda_status(cudaGetLastError());
}
template <typename T, int DP>
int launch_prefill(Attend p, cudaStream_t s) {
  // What the tensor cores cut off may come to half of a result's rounding for so
  // many tokens (fp16: 2048 times 1.1e-7, of 4.9e-4): above, sums are put aside in
  // between. A place has 256 rows of dim, 1 KB dim, of an SM's share of the
  // workspace: 16 + 9 x 128 (dim + 2) bytes.
  p.most = std::is_same<T, __half>::value ? 1 << 15 : 1 << 18;
  if ((long long)p.cols * p.page > p.most) {
    p.places = (int*)p.meta;
    p.aside = (float*)(p.meta + p.sms);
    const int st = cuda_status(cudaMemsetAsync(p.places, 0, p.sms * sizeof(int), s));
    return st == TT_OK ? launch_tiles<T, DP, true>(p, s) : st;
  }
  return launch_tiles<T, DP, false>(p, s);
}
template <typename T>
int launch_dim(const Attend& p, int sms, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (many_rows(p, sms) && p.dim <= 128 && p.heads <= 65535 && p.batch <= 65535)
      return p.dim <= 64 ? launch_prefill<T, 64>(p, s) : launch_prefill<T, 128>(p, s);
  }
  if (p.dim <= 64) return launch<T, 64>(p, sms, s);
  if (p.dim <= 128) return launch<T, 128>(p, sms, s);
  if (p.dim <= 192) return launch<T, 192>(p, sms, s);
  return launch<T, 256>(p, sms, s);
}

}  // namespace
}  // namespace kv8
}  // namespace tt

extern "C" {

size_t tt_kv8_attention_workspace_bytes(int dim) {
  using namespace tt;
  int dev = 0;
  if (dim < 16 || dim > 256 || dim % 16 || check_device(&dev) != TT_OK || kv8::setup(dev) != TT_OK) return 0;
  return kv8::workspace_bytes(dim, kv8::g_sms[dev]);
}

int tt_kv8_attention(const void* q, int type, long long q_stride_b, long long q_stride_s, long long q_stride_h,
                     const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales,
                     const int* block_table, long long table_stride, int columns, const int* lengths,
                     const int* n_query, const float* scale, int causal, void* out, void* workspace,
                     size_t workspace_bytes, int* status, int batch, int S, int heads_q, int heads, int dim,
                     int page, int pages, void* stream) {
  using namespace tt;
  if (!q || !k_codes || !v_codes || !k_scales || !v_scales || !block_table || !lengths || !scale || !out ||
      !workspace || !status)
    return TT_ERR_NULL;
  if (batch <= 0 || S <= 0 || columns <= 0 || heads <= 0 || heads_q <= 0 || heads_q % heads) return TT_ERR_SHAPE;
  if (type < 0 || type > 2 || pages <= 0 || dim < 16 || dim > 256 || dim % 16) return TT_ERR_SHAPE;
  if (page != 16 && page != 32 && page != 64 && page != 128) return TT_ERR_SHAPE;
  const long long rows = (long long)S * (heads_q / heads);
  if (rows > 0x7fffff00LL || (long long)columns * page > 0x7fffff00LL) return TT_ERR_SHAPE;
  const int per = type == q4::kF32 ? 4 : 8;  // values in 16 bytes
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_codes) || !aligned16(v_codes) || !aligned16(workspace) ||
      q_stride_b % per || q_stride_s % per || q_stride_h % per)
    return TT_ERR_ALIGN;
  int dev = 0;
  int st = check_device(&dev);
  if (st != TT_OK) return st;
  if ((st = kv8::setup(dev)) != TT_OK) return st;
  const int sms = kv8::g_sms[dev];
  if (workspace_bytes < kv8::workspace_bytes(dim, sms)) return TT_ERR_WORKSPACE;
  kv8::Attend p;
  p.q = q; p.q_b = q_stride_b; p.q_s = q_stride_s; p.q_h = q_stride_h;
  p.o = out;
  p.kc = (const unsigned char*)k_codes; p.vc = (const unsigned char*)v_codes;
  p.ks = k_scales; p.vs = v_scales;
  p.table = block_table; p.table_b = table_stride; p.lengths = lengths; p.n_query = n_query;
  p.meta = (int4*)workspace;
  p.joint = (float*)((char*)workspace + (size_t)sms * 16);
  p.part = (float*)((char*)p.joint + sms * kv8::piece_bytes(dim));
  p.status = status;
  p.scale = *scale * 1.4426950408889634f;
  p.causal = causal;
  p.batch = batch; p.S = S; p.heads_q = heads_q; p.heads = heads; p.dim = dim; p.page = page; p.pages = pages;
  p.page_log = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  p.cols = columns;
  p.sms = sms;
  p.most = 0;
  p.places = nullptr;
  p.aside = nullptr;
  p.rows = (int)rows;
  cudaStream_t s = (cudaStream_t)stream;
  if (type == q4::kF32) return kv8::launch_dim<float>(p, sms, s);
  if (type == q4::kBF16) return kv8::launch_dim<__nv_bfloat16>(p, sms, s);
  return kv8::launch_dim<__half>(p, sms, s);
}

}  // extern "C"
