// C ABI of microscaled 4-bit floating point and of the experts for a few tokens: argument validation and launches.
// The declarations and the contract of every entry point are in include/dlblas_mxfp4.h.
#include "../../include/dlblas_mxfp4.h"

#include "dispatch.h"
#include "few_rows.h"
#include "mxfp4.h"

namespace dlb {
namespace {

int check_columns(int64_t K) {
  if (K % kMxGroup != 0) return fail(DLB_ERR_BAD_SHAPE, "K=%lld is not a multiple of 32, the columns of a scale", (long long)K);
  if (K > DLB_MXFP4_MAX_COLUMNS) return fail(DLB_ERR_BAD_SHAPE, "K=%lld is beyond %d", (long long)K, DLB_MXFP4_MAX_COLUMNS);
  return DLB_OK;
}

// How a product runs.  us of M x N x K, one side of a border and the other:
//   16 x 2112 x 7168    split 1 x 1: 5.8, 1 x 2: 7.5        16 x 7168 x 18432: 23.0, 16.4
//   17 x 7168 x 18432   split 1 x 2: 29,  2 x 2: 18
//   65 x 2112 x 7168    split 2 x 2: 8.1, 64 tiles: 14.7    128 x 2112 x 7168 (264 workgroups): 13.8, 14.8   65 x 7168 x 18432: 49, 33
//   64 x 7168 x 18432   split 4 x 2: 28,  64 tiles: 32      65: 50, 33
//   256 x 7168 x 18432  64 tiles: 48, 128 tiles: 56         512: 93, 60;  1024 x 2112 x 7168: 28, 26
//   1024 x 7168 x 18432 128 tiles: 104, 256 tiles: 115      2048: 205, 130;  2048 x 2112 x 7168: 39, 50;  4096: 66, 52
enum class MxWay { kSplit11, kSplit12, kSplit22, kSplit42, kTiles64, kTiles128, kTiles256 };
MxWay mx_way(int64_t M, int64_t N) {
  const auto tiles = [&](int m, int n) { return ceil_div(M, m) * ceil_div(N, n); };
  if (M <= 16) return N <= 4096 ? MxWay::kSplit11 : MxWay::kSplit12;
  if (M <= 32 || tiles(32, 32) <= 256) return MxWay::kSplit22;  // workgroups for every CU
  if (M <= 64) return MxWay::kSplit42;
  if (tiles(64, 64) <= 512) return MxWay::kTiles64;  // two a CU
  return tiles(256, 256) >= 128 ? MxWay::kTiles256 : MxWay::kTiles128;
}
// The largest tiles read the scales of four groups at a time: rows of another number of them are laid out anew.
bool mx_pads(int64_t M, int64_t N, int64_t K) { return mx_way(M, N) == MxWay::kTiles256 && K / kMxGroup % 4 != 0; }
int64_t padded(int64_t G) { return ceil_div(G, 4) * 4; }

// Tiles of BM x BN; at most as many workgroups as a launch has threads for.
int mx_tiles(MxArgs& a, int BM, int BN, int threads) {
  const int64_t tiles_m = ceil_div(a.M, BM), tiles_n = ceil_div(a.N, BN);
  if (tiles_m * (tiles_n + 7) > ((1ll << 32) - 1) / threads) return fail(DLB_ERR_BAD_SHAPE, "M=%lld x N=%d beyond the supported range", (long long)a.M, a.N);
  a.tiles_m = static_cast<int>(tiles_m), a.tiles_n = static_cast<int>(tiles_n), a.group_m = static_cast<int>(std::min<int64_t>(tiles_m, 8));
  return DLB_OK;
}

template <class Split>
int launch_split(MxArgs a, hipStream_t st) {
  if (int rc = mx_tiles(a, 16 * Split::MT, 16 * Split::NT, 64 * Split::WAVES)) return rc;
  const dim3 grid(static_cast<unsigned>(ceil_div(a.tiles_n, 8) * 8 * a.tiles_m));
  hipLaunchKernelGGL(mxfp4_split_kernel<Split>, grid, dim3(64 * Split::WAVES), Split::LDS, st, a);
  return finish("mxfp4_gemm");
}

template <class Tile>
int launch_tiles(MxArgs a, hipStream_t st) {
  if (int rc = mx_tiles(a, Tile::BM, Tile::BN, 64 * Tile::WAVES)) return rc;
  with_flag(a.G % 4 != 0, [&](auto ragged) {
    hipLaunchKernelGGL((mxfp4_tile_kernel<Tile, ragged()>), dim3(static_cast<unsigned>(a.tiles_m * a.tiles_n)), dim3(64 * Tile::WAVES), Tile::LDS, st, a);
  });
  return finish("mxfp4_gemm");
}

}  // namespace
}  // namespace dlb

extern "C" {

int dlb_mxfp4_quant(const void* x, int64_t x_row_stride, int dtype, void* q, void* s, int64_t rows, int64_t K, void* stream) {
  using namespace dlb;
  clear_error();
  if (bad_dtype(dtype)) return fail(DLB_ERR_BAD_DTYPE, "dtype %d is not DLB_IN_BF16 / F16 / F32", dtype);
  if (rows < 0 || K < 0) return fail(DLB_ERR_BAD_SHAPE, "negative dimension (rows=%lld K=%lld)", (long long)rows, (long long)K);
  if (int rc = check_columns(K)) return rc;
  if (rows > (1ll << 31) - 1) return fail(DLB_ERR_BAD_SHAPE, "rows=%lld beyond the supported range", (long long)rows);
  if (rows == 0 || K == 0) return DLB_OK;
  if (!x || !q || !s) return fail(DLB_ERR_NULL_POINTER, "x, q or s is NULL");
  if (x_row_stride < 0) return fail(DLB_ERR_BAD_STRIDE, "negative row stride");
  if (off_elements(x, dtype) || misaligned(q, 4)) return fail(DLB_ERR_ALIGNMENT, "x must be aligned to its elements, q to 4 bytes");
  const MxQuantArgs a{x, static_cast<uint32_t*>(q), static_cast<uint8_t*>(s), rows, x_row_stride, static_cast<int>(K)};
  with_type(dtype, [&](auto t) { hipLaunchKernelGGL(mxfp4_quant_kernel<t()>, row_grid(ceil_div(rows * (K / 8), 256)), dim3(256), 0, static_cast<hipStream_t>(stream), a); });
  return finish("mxfp4_quant");
}

size_t dlb_mxfp4_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || !dlb::mx_pads(M, N, K)) return 0;
  return static_cast<size_t>(M + N) * dlb::padded(K / dlb::kMxGroup);
}

int dlb_mxfp4_gemm(const void* a, const void* b, const void* a_s, const void* b_s, void* c, int64_t M, int64_t N, int64_t K, int out_dtype,
                   void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dlb;
  clear_error();
  if (bad_dtype(out_dtype)) return fail(DLB_ERR_BAD_DTYPE, "out_dtype %d is not DLB_IN_BF16 / F16 / F32", out_dtype);
  if (M < 0 || N < 0 || K < 0) return fail(DLB_ERR_BAD_SHAPE, "negative dimension (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
  if (int rc = check_columns(K)) return rc;
  if (M > (1ll << 31) - 1 || N > (1 << 27)) return fail(DLB_ERR_BAD_SHAPE, "M=%lld / N=%lld beyond the supported range", (long long)M, (long long)N);
  if (M == 0 || N == 0) return DLB_OK;
  if (K == 0) return fail(DLB_ERR_BAD_SHAPE, "K=0: there is no product");
  if (!a || !b || !a_s || !b_s || !c) return fail(DLB_ERR_NULL_POINTER, "a, b, a_s, b_s or c is NULL");
  if (misaligned(a, 16) || misaligned(b, 16) || misaligned(a_s, 4) || misaligned(b_s, 4) || off_elements(c, out_dtype))
    return fail(DLB_ERR_ALIGNMENT, "codes must be 16-byte, scales 4-byte aligned, c to its elements");
  const size_t need = dlb_mxfp4_gemm_workspace_bytes(M, N, K);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(DLB_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
  if (need > 0 && misaligned(workspace, 16)) return fail(DLB_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  MxArgs p{};
  p.a = static_cast<const uint8_t*>(a), p.b = static_cast<const uint8_t*>(b), p.a_s = static_cast<const uint8_t*>(a_s), p.b_s = static_cast<const uint8_t*>(b_s);
  p.c = c, p.M = M, p.N = static_cast<int>(N), p.K = static_cast<int>(K), p.G = static_cast<int>(K / kMxGroup), p.pitch = p.G, p.out = out_dtype;
  switch (mx_way(M, N)) {
    case MxWay::kSplit11: return launch_split<MxSplit<1, 1, 8>>(p, st);
    case MxWay::kSplit12: return launch_split<MxSplit<1, 2, 4>>(p, st);
    case MxWay::kSplit22: return launch_split<MxSplit<2, 2, 8>>(p, st);
    case MxWay::kSplit42: return launch_split<MxSplit<4, 2, 4>>(p, st);
    case MxWay::kTiles64: return launch_tiles<MxTile<2, 1, 2, 4>>(p, st);
    case MxWay::kTiles128: return launch_tiles<MxTile<2, 2, 4, 4>>(p, st);
    case MxWay::kTiles256: break;
  }
  if (need > 0) {
    const int words = static_cast<int>(padded(p.G) / 4);
    uint32_t* const to = static_cast<uint32_t*>(workspace);
    const MxPadArgs pad{p.a_s, p.b_s, to, to + M * words, M, N, p.G, words};
    hipLaunchKernelGGL(mxfp4_pad_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div((M + N) * words, 256), 2048))), dim3(256), 0, st, pad);
    if (int rc = finish("mxfp4_gemm (scales)")) return rc;
    p.a_s = reinterpret_cast<const uint8_t*>(to), p.b_s = reinterpret_cast<const uint8_t*>(to + M * words), p.pitch = 4 * words;
  }
  if (int rc = mx_tiles(p, MxRing::kTile, MxRing::kTile, 64 * MxRing::kWaves)) return rc;
  with_type(out_dtype, [&](auto t) {
    hipLaunchKernelGGL(mxfp4_ring_kernel<t()>, dim3(static_cast<unsigned>(p.tiles_m * p.tiles_n)), dim3(64 * MxRing::kWaves), MxRing::kLds, st, p);
  });
  return finish("mxfp4_gemm");
}

int dlb_mxfp4_weight_gemm(const void* x, int64_t x_row_stride, int dtype, const void* q, const void* s, void* y, int64_t M, int64_t N, int64_t K,
                          void* stream) {
  using namespace dlb;
  clear_error();
  if (dtype != kInBf16 && dtype != kInF16) return fail(DLB_ERR_BAD_DTYPE, "dtype %d is not DLB_IN_BF16 / F16", dtype);
  if (M < 0 || N < 0 || K < 0) return fail(DLB_ERR_BAD_SHAPE, "negative dimension (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
  if (int rc = check_columns(K)) return rc;
  if (M > (1 << 21) || N > (1 << 23)) return fail(DLB_ERR_BAD_SHAPE, "M=%lld / N=%lld beyond the supported range", (long long)M, (long long)N);
  if (M == 0 || N == 0) return DLB_OK;
  if (K == 0) return fail(DLB_ERR_BAD_SHAPE, "K=0: there is no product");
  if (!x || !q || !s || !y) return fail(DLB_ERR_NULL_POINTER, "x, q, s or y is NULL");
  if (x_row_stride < 0 || x_row_stride > (1 << 23)) return fail(DLB_ERR_BAD_STRIDE, "x row stride %lld is not 0 ... 2^23", (long long)x_row_stride);
  if (misaligned(q, 16) || misaligned(x, 4) || x_row_stride % 2 != 0 || off_elements(y, dtype))
    return fail(DLB_ERR_ALIGNMENT, "q must be 16-byte, rows of x 4-byte aligned, y to its elements");
  const FewArgs a{x, y, M, x_row_stride, Matrix{static_cast<const uint8_t*>(q), s, static_cast<int>(N), static_cast<int>(K)}};
  // As few tiles of columns a workgroup as leave one for each CU: more of them share the rows, whose copies are most of what comes into LDS, and of up to eight rows
  // two are enough.  us with 1, 2, 4 tiles: 16 x 4096 x 7168 9.3, 12.0, 16.5;  16 x 7168 x 18432 30, 23, 33;  32 x 4096 x 7168 16.5, 11.9, 16.2;
  // 64 x 7168 x 18432 94, 71, 57;  8 x 18432 x 7168 31, 26, 32.  Rows: 4 x 7168 x 18432 by four 16.7, by eight 17.4;  8 by eight 19.3, by sixteen 19.5;  8 x 18432 x 7168 26, 31.
  const int rows = M <= 4 ? 4 : M <= 8 ? 8 : 16;
  const auto groups = [&](int tiles) { return ceil_div(M, rows) * ceil_div(N, 16 * tiles); };
  const int nt = groups(1) <= 256 ? 1 : groups(2) <= 256 || rows < 16 ? 2 : 4;
  const int64_t tiles = ceil_div(N, 16 * nt);
  if (ceil_div(tiles, 8) > 65535) return fail(DLB_ERR_BAD_SHAPE, "N=%lld beyond the supported range", (long long)N);
  const dim3 grid(static_cast<unsigned>(8 * ceil_div(M, rows)), static_cast<unsigned>(ceil_div(tiles, 8)));
  with_flag(dtype == kInBf16, [&](auto bf16) {
    const auto launch = [&](auto r, auto n) {
      typedef FewShape<kE2m1, r(), n()> Shape;
      hipLaunchKernelGGL((few_rows_kernel<bf16() ? kInBf16 : kInF16, kE2m1, r(), n()>), grid, dim3(64 * Shape::kWaves), Shape::kLds, static_cast<hipStream_t>(stream), a);
    };
    if (rows == 16) return with_chunks<1, 2, 4>(nt, [&](auto n) { launch(std::integral_constant<int, 16>(), n); });
    with_chunks<4, 8>(rows, [&](auto r) { with_chunks<1, 2>(nt, [&](auto n) { launch(r, n); }); });
  });
  return finish("mxfp4_weight_gemm");
}

size_t dlb_few_token_experts_workspace_bytes(int64_t tokens, int64_t topk, int64_t I) {
  return tokens > 0 && topk > 0 && I > 0 ? static_cast<size_t>(tokens) * topk * I * sizeof(float) : 0;
}

int dlb_few_token_experts(const void* x, int64_t x_row_stride, int dtype, const void* ids, int ids_dtype, int64_t ids_stride_m, int64_t ids_stride_k,
                          const float* weights, int weight_type, const void* up_q, const void* up_s, const void* down_q, const void* down_s, void* out,
                          int64_t tokens, int64_t topk, int64_t experts, int64_t H, int64_t I, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dlb;
  clear_error();
  if (dtype != kInBf16 && dtype != kInF16) return fail(DLB_ERR_BAD_DTYPE, "dtype %d is not DLB_IN_BF16 / F16", dtype);
  if (ids_dtype != DLB_IDX_I32 && ids_dtype != DLB_IDX_I64) return fail(DLB_ERR_BAD_DTYPE, "ids_dtype %d is not DLB_IDX_I32 / I64", ids_dtype);
  if (weight_type != DLB_WEIGHTS_E4M3 && weight_type != DLB_WEIGHTS_MXFP4) return fail(DLB_ERR_BAD_DTYPE, "weight_type %d is not DLB_WEIGHTS_E4M3 / MXFP4", weight_type);
  const bool f4 = weight_type == DLB_WEIGHTS_MXFP4;
  const int64_t unit = f4 ? kMxGroup : kScaleBlock;
  if (tokens < 0 || topk < 0 || experts < 0 || H < 0 || I < 0)
    return fail(DLB_ERR_BAD_SHAPE, "negative dimension (tokens=%lld topk=%lld experts=%lld H=%lld I=%lld)", (long long)tokens, (long long)topk, (long long)experts,
                (long long)H, (long long)I);
  if (tokens > kFewTokens || topk < 1 || topk > kFewTopk || experts < 1 || experts > kFewExperts)
    return fail(DLB_ERR_BAD_SHAPE, "tokens=%lld, topk=%lld, experts=%lld: at most %d, 1 ... %d, 1 ... %d", (long long)tokens, (long long)topk, (long long)experts, kFewTokens,
                kFewTopk, kFewExperts);
  if (H % unit != 0 || I % unit != 0 || I == 0 || H > (1 << 20) || I > (1 << 20))
    return fail(DLB_ERR_BAD_SHAPE, "H=%lld, I=%lld must be multiples of %lld, I at least that, both at most 2^20", (long long)H, (long long)I, (long long)unit);
  if (tokens * topk * I > DLB_FEW_NUMBERS) return fail(DLB_ERR_BAD_SHAPE, "tokens * topk * I=%lld is beyond 2^29", (long long)(tokens * topk * I));
  if (tokens == 0 || H == 0) return DLB_OK;
  if (!x || !ids || !weights || !up_q || !up_s || !down_q || !down_s || !out) return fail(DLB_ERR_NULL_POINTER, "a tensor pointer is NULL");
  if (x_row_stride < 0 || x_row_stride > (1 << 23)) return fail(DLB_ERR_BAD_STRIDE, "x row stride %lld is not 0 ... 2^23", (long long)x_row_stride);
  if (ids_stride_m < 0 || ids_stride_k < 0) return fail(DLB_ERR_BAD_STRIDE, "negative stride");
  if (misaligned(x, 4) || x_row_stride % 2 != 0 || misaligned(ids, ids_dtype == DLB_IDX_I64 ? 8 : 4) || misaligned(weights, 4) || misaligned(up_q, 16) ||
      misaligned(down_q, 16) || (!f4 && (misaligned(up_s, 4) || misaligned(down_s, 4))) || off_elements(out, dtype))
    return fail(DLB_ERR_ALIGNMENT, "weights must be 16-byte, rows of x 4-byte aligned, the others to their elements");
  const size_t need = dlb_few_token_experts_workspace_bytes(tokens, topk, I);
  if (!workspace || workspace_bytes < need) return fail(DLB_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
  if (misaligned(workspace, 4)) return fail(DLB_ERR_ALIGNMENT, "workspace must be 4-byte aligned");
  ExpertArgs a{};
  a.x = x, a.ids = ids, a.weights = weights, a.act = static_cast<float*>(workspace), a.out = out;
  a.up = Matrix{static_cast<const uint8_t*>(up_q), up_s, static_cast<int>(2 * I), static_cast<int>(H)};
  a.down = Matrix{static_cast<const uint8_t*>(down_q), down_s, static_cast<int>(H), static_cast<int>(I)};
  a.up_q = a.down_q = 0;
  if (f4) {
    a.up_q = I * H, a.up_s = 2 * I * (H / kMxGroup), a.down_q = H * (I / 2), a.down_s = H * (I / kMxGroup);
  } else {
    a.up_q = 2 * I * H, a.up_s = ceil_div(2 * I, 128) * (H / 128) * 4, a.down_q = H * I, a.down_s = (H / 128) * (I / 128) * 4;
  }
  a.x_rs = x_row_stride, a.ids_s0 = ids_stride_m, a.ids_s1 = ids_stride_k;
  a.T = static_cast<int>(tokens), a.topk = static_cast<int>(topk), a.E = static_cast<int>(experts), a.H = static_cast<int>(H), a.I = static_cast<int>(I);
  a.ids_is64 = ids_dtype == DLB_IDX_I64;
  const int64_t slots = tokens * topk;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 down_grid(static_cast<unsigned>(ceil_div(H, 16 * kDownTiles)));
  // Tokens of an expert that a workgroup takes at a time; one with more reads the expert's weights again, from the caches, and x for rows without a token is
  // not read.  8 of 32 experts, 4096 x 7168, us e4m3 / e2m1 (with four waves to K): 8 tokens by four 148 / 100, by eight 131 / 110; 16 tokens by eight 146 / 121, by sixteen
  // 163 / 147; 32 tokens by eight 224 / 181, by sixteen 174 / 154.
  // The second product's rows share the LDS with what is on its way of the weights, and a wave makes the parts of its rows anew for every chunk.  us, 7168 x 2048, four tokens a
  // pass on eight waves against eight of them (e4m3 on eight waves, of e2m1 there is room for four): 8 tokens x 8 of 32 experts e4m3 67 / 69, e2m1 61 / 89;  16 tokens of 32
  // experts 103 / 81, 92 / 102;  of 24 (5.3 tokens each) e2m1 90 / 89;  of 16 86 / 79.
  const int64_t named = std::min(experts, slots), mean = slots / named;
  const int up_rows = tokens <= 4 ? 4 : tokens <= 8 || mean <= 4 ? 8 : 16;
  const auto launch = [&](auto kt, auto kw) {
    const auto up = [&](auto r, auto split) {
      typedef UpShape<kw(), r(), split()> Shape;
      const dim3 grid(static_cast<unsigned>(ceil_div(I, Shape::kColumns)), static_cast<unsigned>(named));
      hipLaunchKernelGGL((experts_up_kernel<kt(), kw(), r(), split()>), grid, dim3(64 * kUpWaves), Shape::kLds, st, a);
    };
    with_chunks<4, 8, 16>(up_rows, [&](auto r) {
      // Two waves to K, whose runs are then long against their start and end, while that leaves workgroups for three quarters of the CUs; four otherwise, and with e4m3 weights for eight
      // rows or fewer.  us of both products with two / four, 2 slots a token, 8 experts:
      //   e2m1, H = 2048: 5 tokens, I = 544 (136 workgroups) 22.0 / 21.0, 768 (192) 21.0 / 21.3, 2048 (512) 28.7 / 32.1;  H = 7168: 29.9 / 26.8, 29.1 / 28.6, 45.3 / 45.2
      //         64 tokens, H = 2048: I = 1024 (128) 67.9 / 61.4, 1536 (192) 81.9 / 84.8;  16 tokens x 8 of 32 experts, I = 2048: H = 1024 115 / 138, 4096 149 / 163, 7168 189 / 200
      //   e4m3, 64 tokens: H = 2048: I = 1024 64.9 / 58.9, 1536 77.5 / 79.5, 4096 157 / 164;  5 tokens: H = 2048: I = 2048 30.6 / 31.1;  H = 7168: 52.5 / 49.9
      if constexpr (kw() == kE2m1 || r() == 16) {
        const bool enough = ceil_div(I, UpShape<kw(), r(), 2>::kColumns) * named >= 192;
        with_flag(enough, [&](auto two) { up(r, std::integral_constant<int, two() ? 2 : 4>()); });
      } else {
        up(r, std::integral_constant<int, 4>());
      }
    });
    const auto down = [&](auto t, auto waves) {
      const int64_t lds = experts_down_lds<kw(), t(), waves()>(tokens, topk, experts);
      hipLaunchKernelGGL((experts_down_kernel<kt(), kw(), t(), waves()>), down_grid, dim3(64 * waves()), static_cast<size_t>(lds), st, a);
    };
    constexpr std::integral_constant<int, 2> two;
    constexpr std::integral_constant<int, 4> four;
    constexpr std::integral_constant<int, 8> eight;
    if (tokens <= 2) return down(two, eight);
    if (tokens <= 4 || (tokens <= kDownWideTokens && slots <= (kw() == kE2m1 ? 4 : 3) * named)) return down(four, eight);
    if constexpr (kw() == kE4m3) {
      if (tokens <= kDownWideTokens) return down(eight, eight);
    }
    down(eight, four);
  };
  with_flag(dtype == kInBf16, [&](auto bf16) {
    constexpr std::integral_constant<int, bf16() ? kInBf16 : kInF16> kt;
    if (f4)
      launch(kt, std::integral_constant<int, kE2m1>());
    else
      launch(kt, std::integral_constant<int, kE4m3>());
  });
  return finish("few_token_experts");
}

}  // extern "C"
