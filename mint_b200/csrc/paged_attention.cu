// Attention of single query tokens over a paged key-value cache.
//
// Query i (position pos_i of request row_i) sees keys j in [max(0, pos_i - window), pos_i]:
//   o = sum_j softmax_j(scale * q . k_j - slope_h * (pos_i - j)) v_j
// K and V are read once each, 4 * D bytes per key and KV head for 4 * D * G flops (G query heads share
// a KV head): the bound is HBM bandwidth.
#include <algorithm>
#include <climits>

#include "paged.cuh"

namespace mint {
namespace paged {

struct AttnParams {
  const void* q;  // [N, Hq, D]
  const void* kp;
  const void* vp;
  void* o;
  const int* tables;     // [B, W], row stride tstride
  const int* positions;  // [N]
  const int* rows;       // [N] or null (row i = i)
  const float* slopes;   // [Hq] or null
  uint32_t* status;
  long long tstride, kp_page, kp_head, kp_line, vp_page, vp_head, vp_line;
  int N, B, W, Hq, Hkv, n_pages, page_shift, window;
  float scale_log2;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) attend_kernel(AttnParams p) {
  constexpr int E = D / 32;
  __shared__ float s_o[4][D], s_m[4], s_l[4];
  const int h = blockIdx.x, i = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int hk = h / (p.Hq / p.Hkv);
  const int row = p.rows ? p.rows[i] : i;
  int pos = p.positions[i];
  if (row < 0 || row >= p.B) pos = -1;
  pos = min(pos, (p.W << p.page_shift) - 1);
  const int first = p.window >= 0 ? max(0, pos - p.window) : 0;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = to_f32(static_cast<const T*>(p.q)[(static_cast<long long>(i) * p.Hq + h) * D + e * 32 + lane]);
    acc[e] = 0.f;
  }
  const float slope = p.slopes ? p.slopes[h] * 1.4426950408889634f : 0.f;
  for (int j = first + warp; j <= pos; j += 4) {
    const int page = p.tables[row * p.tstride + (j >> p.page_shift)];
    if (page < 0 || page >= p.n_pages) continue;
    const long long line = j & ((1 << p.page_shift) - 1);
    const T* k = static_cast<const T*>(p.kp) + page * p.kp_page + hk * p.kp_head + line * p.kp_line;
    const T* v = static_cast<const T*>(p.vp) + page * p.vp_page + hk * p.vp_head + line * p.vp_line;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], to_f32(k[e * 32 + lane]), s);
    s = warp_sum(s) * p.scale_log2 - slope * static_cast<float>(pos - j);
    const float mn = fmaxf(m, s), f = exp2f(m - mn), w = exp2f(s - mn);
    l = l * f + w;
    m = mn;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(w, to_f32(v[e * 32 + lane]), acc[e] * f);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][e * 32 + lane] = acc[e];
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w]);
  for (int d = threadIdx.x; d < D; d += 128) {
    float x = 0.f;
    L = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float f = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - M);
      L = fmaf(s_l[w], f, L);
      x = fmaf(s_o[w][d], f, x);
    }
    static_cast<T*>(p.o)[(static_cast<long long>(i) * p.Hq + h) * D + d] = from_f32<T>(L > 0.f ? x / L : 0.f);
  }
}

template <typename T>
void launch_attend(const AttnParams& p, int D, cudaStream_t st) {
  const dim3 grid(p.Hq, p.N);  // (query head, query)
  if (D == 64) {
    attend_kernel<T, 64><<<grid, 128, 0, st>>>(p);
  } else if (D == 128) {
    attend_kernel<T, 128><<<grid, 128, 0, st>>>(p);
  } else {
    attend_kernel<T, 256><<<grid, 128, 0, st>>>(p);
  }
}

}  // namespace paged

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& tables,
                           const at::Tensor& positions, const c10::optional<at::Tensor>& rows, int64_t window,
                           const c10::optional<at::Tensor>& slopes, double scale) {
  check_contig(q, "q");
  check_cuda(tables, "block_tables");
  check_contig(positions, "positions");
  const auto dt = q.scalar_type();
  MINT_CHECK(q.dim() == 3 && (dt == at::kBFloat16 || dt == at::kHalf), "paged_attention takes bf16 or fp16 [N, Hq, D]");
  const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2);
  MINT_CHECK(D == 64 || D == 128 || D == 256, "paged_attention takes heads of 64, 128 or 256");
  MINT_CHECK(kp.dim() == 4 && kp.size(1) >= 1 && Hq >= 1 && Hq % kp.size(1) == 0, "query heads must be a multiple of the KV heads");
  paged::check_pool(kp, "k_pages", dt, kp.size(1), D);
  paged::check_pool(vp, "v_pages", dt, kp.size(1), D);
  MINT_CHECK(kp.sizes() == vp.sizes(), "k_pages and v_pages have different shapes");
  MINT_CHECK(tables.dim() == 2 && tables.scalar_type() == at::kInt && (tables.size(1) <= 1 || tables.stride(1) == 1),
             "block_tables must be int32 [B, W] with contiguous rows");
  MINT_CHECK(positions.scalar_type() == at::kInt && positions.numel() == N, "positions are int32, one per query");
  paged::AttnParams p{};
  if (rows.has_value()) {
    check_contig(*rows, "rows");
    MINT_CHECK(rows->scalar_type() == at::kInt && rows->numel() == N, "rows are int32, one per query");
    p.rows = rows->data_ptr<int>();
  } else {
    MINT_CHECK(tables.size(0) == N, "without rows there is one table row per query");
  }
  if (slopes.has_value()) {
    check_contig(*slopes, "alibi_slopes");
    MINT_CHECK(slopes->scalar_type() == at::kFloat && slopes->numel() == Hq, "alibi_slopes are fp32, one per query head");
    p.slopes = slopes->data_ptr<float>();
  }
  auto o = at::empty_like(q);
  if (N == 0) return o;
  const int shift = paged::shift_of(kp.size(2));
  MINT_CHECK(N < (1 << 24) && Hq < (1 << 16) && tables.size(1) <= (INT_MAX >> shift), "paged_attention sizes");
  c10::cuda::CUDAGuard guard(q.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  p.q = q.data_ptr();
  p.kp = kp.data_ptr();
  p.vp = vp.data_ptr();
  p.o = o.data_ptr();
  p.tables = tables.data_ptr<int>();
  p.positions = positions.data_ptr<int>();
  p.status = status_ptr(q.device().index());
  p.tstride = tables.stride(0);
  p.kp_page = kp.stride(0);
  p.kp_head = kp.stride(1);
  p.kp_line = kp.stride(2);
  p.vp_page = vp.stride(0);
  p.vp_head = vp.stride(1);
  p.vp_line = vp.stride(2);
  p.N = static_cast<int>(N);
  p.B = static_cast<int>(tables.size(0));
  p.W = static_cast<int>(tables.size(1));
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(kp.size(1));
  p.n_pages = static_cast<int>(kp.size(0));
  p.page_shift = shift;
  p.window = static_cast<int>(std::max<int64_t>(-1, std::min<int64_t>(window, INT_MAX)));
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  if (dt == at::kBFloat16) {
    paged::launch_attend<__nv_bfloat16>(p, static_cast<int>(D), stream);
  } else {
    paged::launch_attend<__half>(p, static_cast<int>(D), stream);
  }
  MINT_CUDA_CHECK(cudaGetLastError());
  count_launch();
  return o;
}

}  // namespace mint
