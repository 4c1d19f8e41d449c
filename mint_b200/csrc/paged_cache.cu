// Paged key-value cache: the step plan (block tables, slots and positions from request lengths) and
// the fused QK-norm + rotation + append.
//
// A cache layer is two pools [pages, Hkv, page_size, D] (any strides with contiguous D). Slot s is
// line s % page_size of page s / page_size. Page sizes are powers of two. The reference has a dense
// [B, Tmax, Hkv, D] cache only (mint/kvcache/base.py:4-65).
#include <algorithm>
#include <atomic>
#include <climits>

#include "paged.cuh"

namespace mint {
namespace paged {

constexpr int kPlanThreads = 256;
constexpr int kMaxRequests = 16384;
// Lengths and prefix sums saturate here, far above any cache, so that a corrupt length cannot wrap an
// index: 2 * (2^30 - 1) still fits an int.
constexpr int kLenCap = (1 << 30) - 1;

__device__ __forceinline__ int sat_add(int a, int b) { return min(a + b, kLenCap); }
__device__ __forceinline__ int clamp_len(int n) { return min(max(n, 0), kLenCap); }
__device__ __forceinline__ int pages_of(int tokens, int page_shift) {
  return static_cast<int>((static_cast<unsigned>(tokens) + (1u << page_shift) - 1u) >> page_shift);
}

// largest r in [0, n) with prefix[r] <= i, for a non-decreasing prefix with prefix[0] = 0 <= i
__device__ __forceinline__ int last_not_above(const int* prefix, int n, int i) {
  int lo = 0, hi = n;  // prefix[lo] <= i < prefix[hi] (hi = n stands for the end)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= i) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

struct PlanParams {
  const int* seq;    // [B] tokens already cached
  const int* fresh;  // [B] tokens this step
  int* tables;       // [B, W], row stride tstride
  const int* free_pages;
  const int* free_head;
  int* positions;  // [N]
  int* slots;      // [N]
  int* rows;       // [N]
  int* ends;       // [B]
  int* seq_out;    // [B]
  int* head_out;   // [1]
  uint32_t* status;
  long long tstride;
  int B, W, N, n_free, page_shift;
};

// Every block repeats the prefix sums over the requests (B ints, from L2) and then fills its share of
// the tokens, tables and request rows, so no block waits for another: a token that falls into a page
// handed out in this step reads the page id from the free list, not from the table entry that another
// block writes. A few KB to a few MB move: the bound is the launch and two dependent reads from L2 (lengths,
// then table or free list). In a CUDA graph 32 requests with a
// token each take 3.4 us, 256 prompts of 131 thousand tokens 5.8 us.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PlanParams p) {
  extern __shared__ int s_prefix[];  // [B + 1] tokens before request b, [B + 1] fresh pages before it
  int* s_tok = s_prefix;
  int* s_page = s_prefix + p.B + 1;
  __shared__ int s_warp[2][kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int page_size = 1 << p.page_shift;
  const int per = (p.B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
  bool bad = false;
  int tok = 0, pages = 0;
  for (int b = b0; b < b1; ++b) {
    const int seq = clamp_len(p.seq[b]), add = clamp_len(p.fresh[b]);
    bad |= p.seq[b] != seq || p.fresh[b] != add;
    s_tok[b] = add;
    s_page[b] = pages_of(seq + add, p.page_shift) - pages_of(seq, p.page_shift);
    tok = sat_add(tok, add);
    pages = sat_add(pages, s_page[b]);
  }
  // exclusive prefix of the threads' sums: within the warp, then over the warps (saturating adds of
  // non-negative numbers associate)
  int tok_inc = tok, page_inc = pages;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, tok_inc, d), c = __shfl_up_sync(0xffffffffu, page_inc, d);
    if (lane >= d) {
      tok_inc = sat_add(tok_inc, a);
      page_inc = sat_add(page_inc, c);
    }
  }
  if (lane == 31) {
    s_warp[0][warp] = tok_inc;
    s_warp[1][warp] = page_inc;
  }
  __syncthreads();
  int tok_at = __shfl_up_sync(0xffffffffu, tok_inc, 1), page_at = __shfl_up_sync(0xffffffffu, page_inc, 1);
  if (lane == 0) tok_at = page_at = 0;
  int tok_sum = 0, page_sum = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) {
      tok_at = sat_add(tok_at, s_warp[0][w]);
      page_at = sat_add(page_at, s_warp[1][w]);
    }
    tok_sum = sat_add(tok_sum, s_warp[0][w]);
    page_sum = sat_add(page_sum, s_warp[1][w]);
  }
  for (int b = b0; b < b1; ++b) {
    const int add = s_tok[b], need = s_page[b];
    s_tok[b] = tok_at;
    s_page[b] = page_at;
    tok_at = sat_add(tok_at, add);
    page_at = sat_add(page_at, need);
  }
  if (tid == 0) {
    s_tok[p.B] = tok_sum;
    s_page[p.B] = page_sum;
  }
  __syncthreads();
  const int head = *p.free_head;
  const int left = head < 0 ? 0 : max(0, p.n_free - head);  // pages that can be handed out
  const int page_cap = INT_MAX >> p.page_shift;              // pages whose slots fit an int
  bad |= tok_sum > p.N || page_sum > left || head < 0;
  const int gtid = blockIdx.x * kPlanThreads + tid, gsize = gridDim.x * kPlanThreads;

  for (int i = gtid; i < p.N; i += gsize) {
    int pos = -1, slot = -1, row = -1;
    if (i < tok_sum) {
      row = last_not_above(s_tok, p.B, i);
      const int seq = clamp_len(p.seq[row]);
      pos = seq + i - s_tok[row];
      const int page_no = pos >> p.page_shift;
      const int have = pages_of(seq, p.page_shift);
      int page = -1;
      if (page_no < p.W) {
        if (page_no < have) {
          page = p.tables[row * p.tstride + page_no];
        } else {
          const int k = s_page[row] + page_no - have;
          if (k < left) page = p.free_pages[head + k];
        }
      }
      if (page >= 0 && page <= page_cap) {
        slot = (page << p.page_shift) | (pos & (page_size - 1));
      } else {
        bad = true;
      }
    }
    p.positions[i] = pos;
    p.slots[i] = slot;
    p.rows[i] = row;
  }
  for (int k = gtid; k < page_sum; k += gsize) {
    const int row = last_not_above(s_page, p.B, k);
    const int col = pages_of(clamp_len(p.seq[row]), p.page_shift) + k - s_page[row];
    if (col < p.W) p.tables[row * p.tstride + col] = k < left ? p.free_pages[head + k] : -1;
  }
  for (int b = gtid; b < p.B; b += gsize) {
    p.ends[b] = s_tok[b + 1];
    p.seq_out[b] = clamp_len(p.seq[b]) + clamp_len(p.fresh[b]);
  }
  if (gtid == 0) *p.head_out = head + min(page_sum, left);
  if (bad) record_status(p.status, kStatusBadArgument);
}

constexpr int plan_smem(int64_t requests) { return static_cast<int>(2 * (requests + 1) * sizeof(int)); }

// Raises the kernel's dynamic shared-memory limit to what kMaxRequests take, once per device: the default of 48 KB
// includes the kernel's static arrays, and a limit set for one call could be lowered by another thread's.
void allow_plan_smem(int device) {
  static std::atomic<uint64_t> ready{0};
  if (ready.load(std::memory_order_relaxed) >> device & 1) return;
  check_smem_optin(plan_smem(kMaxRequests), device, "paged_plan");
  MINT_CUDA_CHECK(cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, plan_smem(kMaxRequests)));
  ready.fetch_or(1ull << device, std::memory_order_relaxed);
}

struct AppendParams {
  const void* qkv;  // [N, (Hq + 2 Hkv) * D], row stride qkv_stride
  const float* qs;
  const float* ks;
  const float* cos_t;  // [S, D / 2] or null (no rotation)
  const float* sin_t;
  const int* positions;
  const int* slots;
  void* q;   // [N, Hq, D]
  void* k;   // [N, Hkv, D] or null
  void* v;   // [N, Hkv, D] or null
  void* kp;  // pools
  void* vp;
  uint32_t* status;
  long long qkv_stride, kp_page, kp_head, kp_line, vp_page, vp_head, vp_line;
  int N, Hq, Hkv, table_len, page_shift, n_pages;
  float eps;
};

// D / 16 lanes own a head row: lane l holds elements 8l .. 8l+7 and, 16 bytes each as well, their rotation
// partners D / 2 further on, so the rotation needs no exchange and 8 cosines and sines serve 16 elements. Norm
// and rotation in fp32, rounded once on the store.
template <typename T, int D>
struct HeadRow {
  static constexpr int L = D / 16;
  uint4 lo, hi;

  __device__ __forceinline__ void load(const T* row) {
    lo = *reinterpret_cast<const uint4*>(row);
    hi = *reinterpret_cast<const uint4*>(row + D / 2);
  }
  __device__ __forceinline__ void store(T* row) const {
    *reinterpret_cast<uint4*>(row) = lo;
    *reinterpret_cast<uint4*>(row + D / 2) = hi;
  }
  // all lanes of the warp call it (the sum runs over the row's L lanes); w = 1 + scale of the two halves
  __device__ __forceinline__ void norm_rotate(const float2 (&w)[2][4], const float2 (&c)[4], const float2 (&sn)[4],
                                              float eps) {
    float2 a[4], b[4], sum = make_float2(0.f, 0.f), sum2 = make_float2(0.f, 0.f);
    unpack8<T>(lo, a);
    unpack8<T>(hi, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sum = ffma2(a[e], a[e], sum);
      sum2 = ffma2(b[e], b[e], sum2);
    }
    sum = fadd2(sum, sum2);
    float ss = sum.x + sum.y;
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    const float norm = rsqrtf(ss * (1.f / D) + eps);
    const float2 n2 = make_float2(norm, norm), minus = make_float2(-norm, -norm);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = fmul2(a[e], w[0][e]), y = fmul2(b[e], w[1][e]);
      a[e] = ffma2(fmul2(x, c[e]), n2, fmul2(fmul2(y, sn[e]), minus));
      b[e] = fmul2(ffma2(x, sn[e], fmul2(y, c[e])), n2);
    }
    lo = pack8<T>(a);
    hi = pack8<T>(b);
  }
};

struct Place {  // where a token goes
  bool known, stored;
  long long page, line;
};
__device__ __forceinline__ Place place_of(const AppendParams& p, int pos, int slot, bool report) {
  Place t;
  t.known = pos >= 0 && (p.cos_t == nullptr || pos < p.table_len);
  const bool in_pool = slot >= 0 && (slot >> p.page_shift) < p.n_pages;
  t.stored = t.known && in_pool;
  t.page = slot >> p.page_shift;
  t.line = slot & ((1 << p.page_shift) - 1);
  if (report && ((pos >= 0 && !t.known) || (slot >= 0 && !in_pool))) record_status(p.status, kStatusBadArgument);
  return t;
}

// 1 + scale of a q or k row's two halves
template <int D>
__device__ __forceinline__ void load_scale(const AppendParams& p, bool is_q, int hl, float2 (&w)[2][4]) {
  const float* scale = (is_q ? p.qs : p.ks) + hl * 8;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    load8(scale + h * (D / 2), w[h]);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[h][e] = make_float2(w[h][e].x + 1.f, w[h][e].y + 1.f);
  }
}

template <int D>
__device__ __forceinline__ void load_turn(const AppendParams& p, int pos, int hl, float2 (&c)[4], float2 (&sn)[4]) {
  if (p.cos_t != nullptr) {
    const long long at = static_cast<long long>(pos) * (D / 2) + hl * 8;
    load8(p.cos_t + at, c);
    load8(p.sin_t + at, sn);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = make_float2(1.f, 1.f), sn[e] = make_float2(0.f, 0.f);
  }
}

template <typename T, int D>
__device__ __forceinline__ void write_row(const AppendParams& p, const Place& t, HeadRow<T, D>& x, int m, int r, int hl) {
  if (!t.known) x.lo = x.hi = make_uint4(0, 0, 0, 0);
  if (r < p.Hq) {
    x.store(static_cast<T*>(p.q) + (static_cast<long long>(m) * p.Hq + r) * D + hl * 8);
    return;
  }
  const bool is_v = r >= p.Hq + p.Hkv;
  const int hk = is_v ? r - p.Hq - p.Hkv : r - p.Hq;
  T* dense = static_cast<T*>(is_v ? p.v : p.k);
  if (dense != nullptr) x.store(dense + (static_cast<long long>(m) * p.Hkv + hk) * D + hl * 8);
  if (t.stored)
    x.store((is_v ? static_cast<T*>(p.vp) + t.page * p.vp_page + hk * p.vp_head + t.line * p.vp_line
                  : static_cast<T*>(p.kp) + t.page * p.kp_page + hk * p.kp_head + t.line * p.kp_line) + hl * 8);
}

// A group of lanes takes ROWS consecutive rows (heads) of one token: all their loads are issued before the
// first reduction, and position, slot, cosines and sines are read once for them. The floor is one read and one
// write of every row; 65536 tokens of 16 + 8 heads of 128 take 149 us in a CUDA graph (5.4 TB/s, 82 % of a plain copy;
// copying the rows to the same places without the arithmetic takes 121 us) and 152 to 164 us as eager calls; with k and
// v returned as well 166 us (86 %). What is left is waiting: cosines are read
// after the position, with 28 warps per SM to hide it. Measured and dropped: four rows per group (163 us, fewer
// warps), persistent warps fed by bulk copies into shared memory (150 us, and far slower for narrow tokens).
// Few tokens are bound by those two dependent reads: 1 token 2.4 us, 64 tokens 2.4 us.
//
// ROWS is 1 below 3 MB of tokens, where more groups hide the latency better, and 2 above (16 + 8 heads: 2 MB 2.9
// against 3.3 us, 4 MB 4.1 against 3.8 us, 256 MB 139 against 104 us).
constexpr int kAppendThreads = 64;
constexpr int64_t kTwoRowsBytes = 3 << 20;

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kAppendThreads, ROWS == 1 ? 1 : 16) append_kernel(AppendParams p) {
  using Row = HeadRow<T, D>;
  const int hl = threadIdx.x % Row::L;
  const int H = p.Hq + 2 * p.Hkv;
  const int units = (H + ROWS - 1) / ROWS;  // per token
  const unsigned unit = blockIdx.x * (kAppendThreads / Row::L) + threadIdx.x / Row::L;
  // lanes past the end repeat the last token's first rows and store nothing: every lane takes part in the sums
  const bool live = unit < static_cast<unsigned>(p.N) * units;
  const int m = live ? unit / units : p.N - 1;
  const int r0 = live ? (unit - m * units) * ROWS : 0;
  const T* src = static_cast<const T*>(p.qkv) + m * p.qkv_stride + hl * 8;
  Row x[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) x[u].load(src + min(r0 + u, H - 1) * D);
  const int pos = p.positions[m], slot = p.slots[m];
  float2 w[2][4], c[4], sn[4];
  if (ROWS == 1) load_scale<D>(p, r0 < p.Hq, hl, w);
  const Place t = place_of(p, pos, slot, live && r0 == 0 && hl == 0);
  load_turn<D>(p, t.known ? pos : 0, hl, c, sn);
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int r = r0 + u;
    const Row raw = x[u];
    if (ROWS > 1) load_scale<D>(p, r < p.Hq, hl, w);
    x[u].norm_rotate(w, c, sn, p.eps);
    if (r >= p.Hq + p.Hkv) x[u] = raw;
    if (live && r < H) write_row<T, D>(p, t, x[u], m, r, hl);
  }
}

template <typename T, int D, int ROWS>
void launch_append(const AppendParams& p, cudaStream_t st) {
  const int64_t units = static_cast<int64_t>(p.N) * ((p.Hq + 2 * p.Hkv + ROWS - 1) / ROWS);
  constexpr int kPerBlock = kAppendThreads / (D / 16);
  append_kernel<T, D, ROWS><<<static_cast<unsigned>((units + kPerBlock - 1) / kPerBlock), kAppendThreads, 0, st>>>(p);
}

template <typename T, int D>
void launch_append(const AppendParams& p, cudaStream_t st) {
  if (static_cast<int64_t>(p.N) * (p.Hq + 2 * p.Hkv) * D * 2 < kTwoRowsBytes) {
    launch_append<T, D, 1>(p, st);
  } else {
    launch_append<T, D, 2>(p, st);
  }
}

template <typename T>
void launch_append(const AppendParams& p, int64_t D, cudaStream_t st) {
  if (D == 64) {
    launch_append<T, 64>(p, st);
  } else if (D == 128) {
    launch_append<T, 128>(p, st);
  } else {
    launch_append<T, 256>(p, st);
  }
}

}  // namespace paged

// Plan of one step over B requests: hands out pages from free_pages[free_head ...] to requests whose
// seq + fresh tokens need more than they have (written into `tables`), and returns positions, slots and
// request rows of the n_tokens packed tokens (-1 beyond the last), the requests' token ends, their new
// lengths and the new head of the free list.
std::vector<at::Tensor> paged_plan(const at::Tensor& seq, const at::Tensor& fresh, at::Tensor& tables,
                                   const at::Tensor& free_pages, const at::Tensor& free_head, int64_t page_size,
                                   int64_t n_tokens) {
  check_contig(seq, "seq_lens");
  check_contig(fresh, "new_lens");
  check_cuda(tables, "block_tables");
  check_contig(free_pages, "free_pages");
  check_contig(free_head, "free_head");
  for (const at::Tensor* t : {&seq, &fresh, static_cast<const at::Tensor*>(&tables), &free_pages, &free_head})
    MINT_CHECK(t->scalar_type() == at::kInt && t->device() == seq.device(), "paged_plan takes int32 tensors on one device");
  const int64_t B = seq.numel();
  MINT_CHECK(fresh.numel() == B && tables.dim() == 2 && tables.size(0) == B && (tables.size(1) <= 1 || tables.stride(1) == 1),
             "paged_plan: one length pair and one table row per request");
  MINT_CHECK(B <= paged::kMaxRequests, "paged_plan takes at most ", paged::kMaxRequests, " requests");
  MINT_CHECK(free_head.numel() == 1, "free_head has one element");
  MINT_CHECK(n_tokens >= 0 && n_tokens <= paged::kLenCap && tables.size(1) < (1ll << 31) && free_pages.numel() < (1ll << 31),
             "paged_plan sizes");
  // one allocation for the outputs; each starts on a 16-byte boundary
  auto round4 = [](int64_t n) { return (n + 3) / 4 * 4; };
  const int64_t nt = round4(n_tokens), nb = round4(B);
  auto out = paged::empty_cuda({3 * nt + 2 * nb + 4}, at::kInt, seq.device());
  std::vector<at::Tensor> views{paged::flat_view(out, 0, n_tokens),      paged::flat_view(out, nt, n_tokens), paged::flat_view(out, 2 * nt, n_tokens),
                                paged::flat_view(out, 3 * nt, B),        paged::flat_view(out, 3 * nt + nb, B), paged::flat_view(out, 3 * nt + 2 * nb, 1)};
  c10::cuda::CUDAGuard guard(seq.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  paged::PlanParams p{};
  p.seq = seq.data_ptr<int>();
  p.fresh = fresh.data_ptr<int>();
  p.tables = tables.data_ptr<int>();
  p.free_pages = free_pages.data_ptr<int>();
  p.free_head = free_head.data_ptr<int>();
  p.positions = out.data_ptr<int>();
  p.slots = p.positions + nt;
  p.rows = p.slots + nt;
  p.ends = p.rows + nt;
  p.seq_out = p.ends + nb;
  p.head_out = p.seq_out + nb;
  p.status = status_ptr(seq.device().index());
  p.tstride = tables.stride(0);
  p.B = static_cast<int>(B);
  p.W = static_cast<int>(tables.size(1));
  p.N = static_cast<int>(n_tokens);
  p.n_free = static_cast<int>(free_pages.numel());
  p.page_shift = paged::shift_of(page_size);
  const int smem = paged::plan_smem(B);
  paged::allow_plan_smem(seq.device().index());
  const int64_t work = std::max<int64_t>(n_tokens, B);
  const int grid = static_cast<int>(std::min<int64_t>(std::max<int64_t>((work + 1023) / 1024, 1), num_sms(seq.device().index())));
  paged::plan_kernel<<<grid, paged::kPlanThreads, smem, stream>>>(p);
  MINT_CUDA_CHECK(cudaGetLastError());
  count_launch();
  return views;
}

// q [N, Hq, D] normed and rotated; k (normed, rotated) and v stored into the pools' slots. With `dense`
// also returns k and v as [N, Hkv, D].
std::vector<at::Tensor> qk_norm_rope_paged(const at::Tensor& qkv, int64_t n_q, int64_t n_kv, int64_t D,
                                           const at::Tensor& qs, const at::Tensor& ks,
                                           const c10::optional<at::Tensor>& cos_t,
                                           const c10::optional<at::Tensor>& sin_t, const at::Tensor& positions,
                                           const at::Tensor& slots, at::Tensor& kp, at::Tensor& vp, double eps,
                                           bool dense) {
  paged::check_inference("qk_norm_rope_paged", {&qkv, &qs, &ks, &kp, &vp});
  if (cos_t.has_value()) paged::check_inference("qk_norm_rope_paged", {&*cos_t});
  if (sin_t.has_value()) paged::check_inference("qk_norm_rope_paged", {&*sin_t});
  check_cuda(qkv, "qkv");
  check_contig(positions, "positions");
  check_contig(slots, "slots");
  check_contig(qs, "q_scale");
  check_contig(ks, "k_scale");
  const auto dt = qkv.scalar_type();
  MINT_CHECK((dt == at::kBFloat16 || dt == at::kHalf) && (D == 64 || D == 128 || D == 256),
             "qk_norm_rope_paged takes bf16 or fp16 heads of 64, 128 or 256");
  MINT_CHECK(n_q >= 1 && n_kv >= 1 && qkv.dim() == 2 && qkv.size(1) == (n_q + 2 * n_kv) * D, "qkv must be [N, ",
             (n_q + 2 * n_kv) * D, "]");
  MINT_CHECK(qkv.stride(1) == 1 && (qkv.size(0) <= 1 || qkv.stride(0) % 8 == 0) && reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0,
             "qkv rows must be contiguous and 16-byte aligned");
  const int64_t N = qkv.size(0);
  MINT_CHECK(positions.scalar_type() == at::kInt && slots.scalar_type() == at::kInt && positions.numel() == N &&
                 slots.numel() == N,
             "positions and slots are int32, one per token");
  MINT_CHECK(qs.scalar_type() == at::kFloat && ks.scalar_type() == at::kFloat && qs.numel() == D && ks.numel() == D,
             "norm scales are fp32 [head_dim]");
  paged::check_vec16(qs, "q_scale");
  paged::check_vec16(ks, "k_scale");
  paged::check_pool(kp, "k_pages", dt, n_kv, D);
  paged::check_pool(vp, "v_pages", dt, n_kv, D);
  MINT_CHECK(kp.sizes() == vp.sizes(), "k_pages and v_pages have different shapes");
  for (const at::Tensor* t : {&positions, &slots, &qs, &ks, static_cast<const at::Tensor*>(&kp), static_cast<const at::Tensor*>(&vp)})
    MINT_CHECK(t->device() == qkv.device(), "qk_norm_rope_paged takes tensors on one device");
  paged::AppendParams p{};
  if (cos_t.has_value()) {
    MINT_CHECK(sin_t.has_value(), "rotation needs both cos and sin");
    check_contig(*cos_t, "cos");
    check_contig(*sin_t, "sin");
    MINT_CHECK(cos_t->scalar_type() == at::kFloat && sin_t->scalar_type() == at::kFloat && cos_t->dim() == 2 &&
                   cos_t->size(0) >= 1 && cos_t->size(1) == D / 2 && cos_t->sizes() == sin_t->sizes(),
               "cos / sin are fp32 [positions, head_dim / 2] with one position at least");
    paged::check_vec16(*cos_t, "cos");
    paged::check_vec16(*sin_t, "sin");
    MINT_CHECK(cos_t->device() == qkv.device() && sin_t->device() == qkv.device(), "qk_norm_rope_paged takes tensors on one device");
    p.cos_t = cos_t->data_ptr<float>();
    p.sin_t = sin_t->data_ptr<float>();
    p.table_len = static_cast<int>(std::min<int64_t>(cos_t->size(0), INT32_MAX));
  }
  auto q = paged::empty_cuda({N, n_q, D}, dt, qkv.device());
  std::vector<at::Tensor> out{q};
  if (dense) {
    out.push_back(paged::empty_cuda({N, n_kv, D}, dt, qkv.device()));
    out.push_back(paged::empty_cuda({N, n_kv, D}, dt, qkv.device()));
  }
  if (N == 0) return out;
  MINT_CHECK(N * (n_q + 2 * n_kv) < (1ll << 31), "qk_norm_rope_paged: too many rows for one call");
  c10::cuda::CUDAGuard guard(qkv.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  p.qkv = qkv.data_ptr();
  p.qs = qs.data_ptr<float>();
  p.ks = ks.data_ptr<float>();
  p.positions = positions.data_ptr<int>();
  p.slots = slots.data_ptr<int>();
  p.q = q.data_ptr();
  p.k = dense ? out[1].data_ptr() : nullptr;
  p.v = dense ? out[2].data_ptr() : nullptr;
  p.kp = kp.data_ptr();
  p.vp = vp.data_ptr();
  p.status = status_ptr(qkv.device().index());
  p.qkv_stride = qkv.stride(0);
  p.kp_page = kp.stride(0);
  p.kp_head = kp.stride(1);
  p.kp_line = kp.stride(2);
  p.vp_page = vp.stride(0);
  p.vp_head = vp.stride(1);
  p.vp_line = vp.stride(2);
  p.N = static_cast<int>(N);
  p.Hq = static_cast<int>(n_q);
  p.Hkv = static_cast<int>(n_kv);
  p.page_shift = paged::shift_of(kp.size(2));
  p.n_pages = static_cast<int>(kp.size(0));
  p.eps = static_cast<float>(eps);
  if (dt == at::kBFloat16) {
    paged::launch_append<__nv_bfloat16>(p, D, stream);
  } else {
    paged::launch_append<__half>(p, D, stream);
  }
  MINT_CUDA_CHECK(cudaGetLastError());
  count_launch();
  return out;
}

}  // namespace mint
