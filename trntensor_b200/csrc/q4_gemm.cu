// Products of many rows with a 4-bit matrix: launches (csrc/q4_gemm.cuh).
#include "common.cuh"
#include "q4_gemm.cuh"
#include "q4_host.cuh"

namespace tt {
namespace q4 {
namespace {

std::once_flag g_flags[kMaxDevices];
int g_ok[kMaxDevices];
int g_sms[kMaxDevices];

template <int R, int MT, int kGroups, bool kTrans, bool kSums>
int set_attr() {
  return cudaFuncSetAttribute(gemm_kernel<R, MT, kGroups, kTrans, kSums>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              GemmShape<R, MT, kSums>::kSmem) == cudaSuccess
             ? TT_OK
             : TT_ERR_CUDA;
}
template <int R, int MT, bool kSums>
int set_attrs() {
  int st = set_attr<R, MT, 1, false, kSums>();
  if (st == TT_OK) st = set_attr<R, MT, 2, false, kSums>();
  if (st == TT_OK) st = set_attr<R, MT, 4, false, kSums>();
  if (st == TT_OK) st = set_attr<R, MT, 1, true, kSums>();
  if (st == TT_OK) st = set_attr<R, MT, 2, true, kSums>();
  if (st == TT_OK) st = set_attr<R, MT, 4, true, kSums>();
  return st;
}
int setup(int dev) {
  return once_per_device(g_flags, g_ok, dev, [dev]() -> int {
    if (cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return TT_ERR_CUDA;
    int st = set_attrs<1, 32, false>();
    if (st == TT_OK) st = set_attrs<1, 64, false>();
    if (st == TT_OK) st = set_attrs<1, 128, false>();
    if (st == TT_OK) st = set_attrs<1, 256, false>();
    if (st == TT_OK) st = set_attrs<2, 256, false>();
    if (st == TT_OK) st = set_attrs<1, 32, true>();
    if (st == TT_OK) st = set_attrs<1, 64, true>();
    if (st == TT_OK) st = set_attrs<1, 128, true>();
    return st;
  });
}

inline size_t al256(size_t x) { return (x + 255) / 256 * 256; }
inline long long pad64(long long x) { return (x + 63) / 64 * 64; }

template <int R, int MT, int kGroups, bool kTrans, bool kSums>
int launch(const CUtensorMap& map, Gemm p, int splits, cudaStream_t s) {
  const long long rows = kTrans ? p.K : p.N;
  p.tiles_m = (p.M + MT - 1) / MT;
  const long long tiles = (rows + R * 128 - 1) / (R * 128) * p.tiles_m;
  cudaLaunchConfig_t cfg = {};
  if (!grid_of(tiles, splits, &cfg.gridDim)) return TT_ERR_SHAPE;
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = GemmShape<R, MT, kSums>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, gemm_kernel<R, MT, kGroups, kTrans, kSums>, map, p));
}
template <int R, int MT, bool kTrans, bool kSums>
int launch_groups(const CUtensorMap& map, const Gemm& p, int group, int splits, cudaStream_t s) {
  if (group == 128) return launch<R, MT, 1, kTrans, kSums>(map, p, splits, s);
  if (group == 64) return launch<R, MT, 2, kTrans, kSums>(map, p, splits, s);
  return launch<R, MT, 4, kTrans, kSums>(map, p, splits, s);
}
template <bool kTrans>
int launch_tile(const CUtensorMap& map, const Gemm& p, int group, int R, int MT, bool sums, int splits, cudaStream_t s) {
  if (sums) {
    if (MT == 32) return launch_groups<1, 32, kTrans, true>(map, p, group, splits, s);
    if (MT == 64) return launch_groups<1, 64, kTrans, true>(map, p, group, splits, s);
    return launch_groups<1, 128, kTrans, true>(map, p, group, splits, s);
  }
  if (R == 2) return launch_groups<2, 256, kTrans, false>(map, p, group, splits, s);
  if (MT == 32) return launch_groups<1, 32, kTrans, false>(map, p, group, splits, s);
  if (MT == 64) return launch_groups<1, 64, kTrans, false>(map, p, group, splits, s);
  if (MT == 128) return launch_groups<1, 128, kTrans, false>(map, p, group, splits, s);
  return launch_groups<1, 256, kTrans, false>(map, p, group, splits, s);
}

template <typename XT>
int convert(const void* x, long long ldx, const float* col, int M, int C, int Cp, int terms, int finite, void* out,
            float* f, cudaStream_t s) {
  const int wide = aligned16(x) && ldx % (16 / (int)sizeof(XT)) == 0;
  if (terms == 2)
    convert_kernel<XT, 2><<<M, 256, 0, s>>>((const XT*)x, ldx, col, M, C, Cp, wide, (__half*)out, f, finite);
  else
    convert_kernel<XT, 1><<<M, 256, 0, s>>>((const XT*)x, ldx, col, M, C, Cp, wide, (__half*)out, f, finite);
  return cuda_status(cudaGetLastError());
}

}  // namespace

size_t gemm_workspace_bytes(int type, int scale_type, bool transposed, int M, int N, int K) {
  const size_t C = transposed ? N : K;
  const int planes = (type == kF32 ? 2 : 1) + (scale_type == kF32 ? 1 : 0);
  return al256((size_t)M * 4) + al256((size_t)planes * M * pad64(C) * 2);
}

int run_gemm(bool transposed, const void* x, int type, long long ldx, const void* packed, const void* scales,
             int scale_type, const float* row_scale, int M, int N, int K, int group, void* y, long long ldy,
             void* workspace, size_t workspace_bytes, int* err, int dev, cudaStream_t s) {
  if (workspace_bytes < gemm_workspace_bytes(type, scale_type, transposed, M, N, K)) return TT_ERR_WORKSPACE;
  if (!aligned16(workspace)) return TT_ERR_ALIGN;
  int st = setup(dev);
  if (st != TT_OK) return st;
  const int sms = g_sms[dev];
  const int C = transposed ? N : K;
  const long long rows = transposed ? K : N;
  Gemm p = {};
  p.packed = (const uint4*)packed;
  p.scales = scales;
  p.scales_f32 = scale_type == kF32;
  p.row_scale = row_scale;
  p.out = y;
  p.type = type;
  p.ldo = ldy;
  p.M = M; p.N = N; p.K = K;
  p.kblocks = (int)(((long long)K + kCols - 1) / kCols);
  p.steps = (int)(((long long)C + 127) / 128);
  p.err = err;
  const int terms = type == kF32 ? 2 : 1;
  // pairs of terms (scale, x) that reach the result's precision
  p.passes = 1;
  if (terms == 2) { p.scale_term[p.passes] = 0; p.x_term[p.passes++] = 1; }
  if (p.scales_f32) { p.scale_term[p.passes] = 1; p.x_term[p.passes++] = terms; }
  if (p.scales_f32 && terms == 2) { p.scale_term[p.passes] = 2; p.x_term[p.passes++] = terms; }

  // the dense operand: fp16 rows are taken as they stand where TMA can read them
  const bool direct = type == kF16 && !p.scales_f32 && !transposed && aligned16(x) && ldx % 8 == 0;
  const void* b = x;
  uint64_t dims[3] = {(uint64_t)C, (uint64_t)M, 1}, strides[2] = {(uint64_t)ldx * 2, (uint64_t)ldx * 2 * M};
  if (!direct) {
    float* f = (float*)workspace;
    void* w = (char*)workspace + al256((size_t)M * 4);
    const int Cp = (int)pad64(C);
    const float* col = transposed ? row_scale : nullptr;
    if (type == kF32) st = convert<float>(x, ldx, col, M, C, Cp, 2, p.scales_f32, w, f, s);
    else if (type == kBF16) st = convert<__nv_bfloat16>(x, ldx, col, M, C, Cp, 1, p.scales_f32, w, f, s);
    else st = convert<__half>(x, ldx, col, M, C, Cp, 1, p.scales_f32, w, f, s);
    if (st != TT_OK) return st;
    p.f = f;
    b = w;
    dims[0] = Cp;
    dims[2] = terms + p.scales_f32;
    strides[0] = (uint64_t)Cp * 2;
    strides[1] = (uint64_t)Cp * 2 * M;
  }
  // Sums that leave the tensor cores in between: for fp32, and for sums so long
  // that what is cut off may come to half of the result's rounding (fp16: 2048
  // times 1.1e-7, of 4.9e-4; bf16 eight times as many).
  const bool sums = type == kF32 || C > (type == kF16 ? 1 << 15 : 1 << 18);
  // Tile: all tokens up to 256 at a time; 256 rows of the matrix where that
  // makes the last wave of CTAs no emptier (time goes by waves times rows).
  // Sums take registers: 128 tokens at most.
  const int MT = M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 || sums ? 128 : 256;
  const long long tiles_m = ((long long)M + MT - 1) / MT;
  const long long one = (rows + 127) / 128 * tiles_m, two = (rows + 255) / 256 * tiles_m;
  const int R = MT == 256 && (two + sms - 1) / sms * 2 <= (one + sms - 1) / sms ? 2 : 1;
  int splits = 1;
  while (R == 1 && splits < 8 && one * splits * 2 <= sms && p.steps >= splits * 4) splits *= 2;
  const uint32_t box[3] = {64, (uint32_t)MT, 1};
  CUtensorMap map;
  if (encode_tmap(&map, b, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_FLOAT16))
    return TT_ERR_TMA;
  return transposed ? launch_tile<true>(map, p, group, R, MT, sums, splits, s)
                    : launch_tile<false>(map, p, group, R, MT, sums, splits, s);
}

int run_row_scale(const void* scales, int scale_type, int N, int K, int group, float* out, cudaStream_t s) {
  const int kblocks = (int)(((long long)K + kCols - 1) / kCols);
  const long long ctas = (((long long)N + kRows - 1) / kRows + 7) / 8;
  if (scale_type == kF32)
    row_scale_kernel<float><<<(unsigned)ctas, 256, 0, s>>>((const float*)scales, N, kblocks, kCols / group, out);
  else
    row_scale_kernel<__nv_bfloat16><<<(unsigned)ctas, 256, 0, s>>>((const __nv_bfloat16*)scales, N, kblocks,
                                                                   kCols / group, out);
  return cuda_status(cudaGetLastError());
}

}  // namespace q4
}  // namespace tt
