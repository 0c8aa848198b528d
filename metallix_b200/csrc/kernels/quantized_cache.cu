// The cache in 8 bits: norm, rotation and the write of keys and values as codes
// in one pass over a step's projections, and pages read back into the compute
// type. The rows are those of quantized.cuh. The reference's pool holds rows in
// the compute type only (crates/models/qwen/src/forward/paged.rs:300-325); this
// is the same write with half the bytes (a quarter of float32's).
#include "quantized.cuh"

namespace mxb {

struct StoreArgs {
  const void *q_in, *k_in, *v_in;
  long long q_stride, k_stride, v_stride;   // row strides in elements
  void* q_out;                              // [tokens, heads, head_dim]; null: no queries
  uint8_t* codes;                           // null: no write
  float* scales;
  const int *slots, *positions;
  const float *q_weight, *k_weight;         // null: no norm
  const float *cos_table, *sin_table;       // null: no rotation
  int table_positions, rotary_dim, interleaved;
  const float* row_sums;                    // [tokens, 2] mean squares of a token's whole q and k; null: the norm is a head's own
  int tokens, heads, kv_heads, head_dim, page_tokens, num_pages;
  float eps;
  const float* q_factors;                   // what queries are multiplied by, per position; null: nothing
  int factor_positions;
  int* status;
};

// Mean squares of each token's query and key projections, for a norm over the whole projection.
template <typename T>
__global__ void __launch_bounds__(256) projection_squares_kernel(const T* __restrict__ q, const T* __restrict__ k, long long q_stride,
                                                                 long long k_stride, int q_width, int k_width, float* __restrict__ out) {
  __shared__ float scratch[33];
  const bool is_k = blockIdx.y != 0;
  const int width = is_k ? k_width : q_width;
  const T* row = is_k ? k + blockIdx.x * k_stride : q + blockIdx.x * q_stride;
  float sum = 0.0f;
  for (int i = threadIdx.x; i < width; i += blockDim.x) {
    const float x = to_float(row[i]);
    sum += x * x;
  }
  sum = block_sum(sum, scratch);
  if (threadIdx.x == 0) out[2 * blockIdx.x + (is_k ? 1 : 0)] = width > 0 ? sum / static_cast<float>(width) : 0.0f;
}

// The general form: a block per (token, head), for every head size and
// rotation. The values of a head go through shared memory, where a value's
// rotation partner is found wherever it lies.
template <typename T, int KIND>
__global__ void __launch_bounds__(256) store_quantized_kernel(const StoreArgs a) {
  extern __shared__ float head[];   // head_dim values
  __shared__ float scratch[33];
  __shared__ uint32_t largest;
  const int t = blockIdx.x, h = blockIdx.y;   // 0..heads-1: q, then kv_heads of k, then kv_heads of v
  const bool is_q = h < a.heads, is_k = !is_q && h < a.heads + a.kv_heads;
  const int kv = is_q ? 0 : (is_k ? h - a.heads : h - a.heads - a.kv_heads);
  const int n = a.head_dim;
  const T* src = is_q   ? static_cast<const T*>(a.q_in) + t * a.q_stride + static_cast<long long>(h) * n
                 : is_k ? static_cast<const T*>(a.k_in) + t * a.k_stride + static_cast<long long>(kv) * n
                        : static_cast<const T*>(a.v_in) + t * a.v_stride + static_cast<long long>(kv) * n;
  size_t pool_row = 0;
  if (is_q) {
    if (a.q_out == nullptr) return;
  } else {
    const int slot = a.slots[t];
    if (slot < 0) return;   // this token does not write the cache
    const int page = slot / a.page_tokens;
    if (page >= a.num_pages) {
      if (threadIdx.x == 0) atomicOr(a.status, kStatusBadSlot);
      return;
    }
    pool_row = ((static_cast<size_t>(page) * 2 + (is_k ? 0 : 1)) * a.kv_heads + kv) * a.page_tokens + (slot - page * a.page_tokens);
  }
  if (threadIdx.x == 0) largest = 0;
  const bool worked = is_q || is_k;   // values are stored as projected
  const float* weight = is_q ? a.q_weight : (is_k ? a.k_weight : nullptr);
  float sum = 0.0f;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const float x = to_float(src[i]);
    head[i] = x;
    sum += x * x;
  }
  if (weight != nullptr) {
    float mean;
    if (a.row_sums != nullptr) {
      mean = a.row_sums[2 * t + (is_k ? 1 : 0)];
      weight += static_cast<size_t>(is_q ? h : kv) * n;
    } else {
      mean = block_sum(sum, scratch) / static_cast<float>(n);
    }
    const float scale = rsqrtf(mean + a.eps);
    for (int i = threadIdx.x; i < n; i += blockDim.x) head[i] = head[i] * scale * weight[i];
  }
  __syncthreads();
  const int half = a.rotary_dim >> 1;
  int pos = a.positions[t];
  float factor = 1.0f;
  if (is_q && a.q_factors != nullptr) {
    const bool there = pos >= 0 && pos < a.factor_positions;
    if (!there && threadIdx.x == 0) atomicOr(a.status, kStatusBadSlot);
    factor = a.q_factors[there ? pos : 0];
  }
  const bool rotate = worked && a.cos_table != nullptr;
  if (rotate && (pos < 0 || pos >= a.table_positions)) {
    if (threadIdx.x == 0) atomicOr(a.status, kStatusBadSlot);
    pos = 0;
  }
  float kept[2];   // at most 512 values a head, 256 threads
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = threadIdx.x + j * static_cast<int>(blockDim.x);
    if (i >= n) continue;
    float out = head[i];
    if (rotate && i < a.rotary_dim) {
      const bool first = a.interleaved ? (i & 1) == 0 : i < half;
      const int pair = a.interleaved ? i >> 1 : (first ? i : i - half);
      const int partner = a.interleaved ? i ^ 1 : (first ? i + half : i - half);
      const float c = a.cos_table[static_cast<size_t>(pos) * half + pair];
      const float s = a.sin_table[static_cast<size_t>(pos) * half + pair];
      out = first ? head[i] * c - head[partner] * s : head[i] * c + head[partner] * s;
    }
    kept[j] = out * factor;
    if (!is_q) atomicMax(&largest, magnitude_bits(out));
  }
  if (is_q) {
    T* dst = static_cast<T*>(a.q_out) + (static_cast<size_t>(t) * a.heads + h) * n;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = threadIdx.x + j * static_cast<int>(blockDim.x);
      if (i < n) dst[i] = from_float<T>(kept[j]);
    }
    return;
  }
  __syncthreads();
  const RowScale row = row_scale<KIND>(largest);
  uint8_t* dst = a.codes + pool_row * n;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = threadIdx.x + j * static_cast<int>(blockDim.x);
    if (i < n) dst[i] = static_cast<uint8_t>(code_of<KIND>(kept[j], row));
  }
  if (threadIdx.x == 0) a.scales[pool_row] = row.scale;
}

// Pages back into the compute type: block (page of the table, request). The
// rows up to the request's last position are written, everything else of
// `out` stays as it is.
template <typename T, int KIND>
__global__ void __launch_bounds__(256)
read_cache_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, T* __restrict__ out,
                  const int* __restrict__ block_tables, int max_pages, const int* __restrict__ row_request,
                  const int* __restrict__ first, const int* __restrict__ last, int kv_heads, int head_dim, int page_tokens,
                  int num_pages, int window, int chunk, int keep, int* status) {
  const int slot = blockIdx.x, row = blockIdx.y;
  const int begin = first_visible_key(max(first[row], 0), window, chunk), end = last[row];
  const int key0 = slot * page_tokens;
  if (key0 > end || (key0 + page_tokens <= begin && key0 >= keep)) return;
  const int page = block_tables[static_cast<size_t>(row_request[row]) * max_pages + slot];
  if (page < 0 || page >= num_pages) {
    if (threadIdx.x == 0) atomicOr(status, kStatusBadPage);
    return;
  }
  const int rows = min(page_tokens, end - key0 + 1);
  const size_t base = static_cast<size_t>(page) * 2 * kv_heads * page_tokens;
  for (int i = threadIdx.x; i < 2 * kv_heads * rows * head_dim; i += blockDim.x) {
    const int line = i / head_dim, d = i - line * head_dim;
    const int head = line / rows, r = line - head * rows;
    const size_t at = base + static_cast<size_t>(head) * page_tokens + r;
    out[at * head_dim + d] = from_float<T>(code_value<KIND>(codes[at * head_dim + d]) * scales[at]);
  }
}

}  // namespace mxb

using namespace mxb;

static bool pool_fits(int num_pages, int kv_heads, int page_tokens) {
  return num_pages > 0 && kv_heads > 0 && page_tokens > 0 &&
         static_cast<long long>(num_pages) * 2 * kv_heads * page_tokens <= 0x7fffffffLL;
}

// The norm and rotation of a step's queries and keys, queries to q_out, keys and
// values into the pool as codes at `slots` (negative: not written). row_sums:
// float32 scratch of 2 * tokens values for norm_scope 1 (a norm over a token's
// whole projection; weights [heads * head_dim] and [kv_heads * head_dim]).
MXB_API int mxb_store_quantized(const void* q_in, const void* k_in, const void* v_in, long long q_stride, long long k_stride,
                                long long v_stride, void* q_out, void* codes, float* scales, int kind, const int* slots,
                                const int* positions, const float* q_weight, const float* k_weight, const float* cos_table,
                                const float* sin_table, int table_positions, int rotary_dim, int interleaved, int norm_scope,
                                float* row_sums, int tokens, int heads, int kv_heads, int head_dim, int page_tokens, int num_pages,
                                float eps, int dtype, const float* q_factors, int factor_positions, int* status,
                                cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (codes == nullptr || scales == nullptr || slots == nullptr || !pool_fits(num_pages, kv_heads, page_tokens) || head_dim <= 0 ||
      head_dim > 512 || heads < 0 || heads + 2 * kv_heads > 65535 || rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1) ||
      (dtype != kF32 && dtype != kBF16) || (kind != kCodesE4M3 && kind != kCodesInt8) || (norm_scope == 1 && row_sums == nullptr))
    return static_cast<int>(cudaErrorInvalidValue);
  if (norm_scope == 1 && (q_weight != nullptr || k_weight != nullptr)) {
    const dim3 grid(tokens, 2);
    if (dtype == kF32)
      projection_squares_kernel<float><<<grid, 256, 0, stream>>>(static_cast<const float*>(q_in), static_cast<const float*>(k_in), q_stride,
                                                                  k_stride, heads * head_dim, kv_heads * head_dim, row_sums);
    else
      projection_squares_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(
          static_cast<const __nv_bfloat16*>(q_in), static_cast<const __nv_bfloat16*>(k_in), q_stride, k_stride, heads * head_dim,
          kv_heads * head_dim, row_sums);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  const StoreArgs args = {q_in, k_in, v_in, q_stride, k_stride, v_stride, q_out, static_cast<uint8_t*>(codes), scales, slots, positions,
                          q_weight, k_weight, cos_table, sin_table, table_positions, rotary_dim, interleaved,
                          norm_scope == 1 ? row_sums : nullptr, tokens, heads, kv_heads, head_dim, page_tokens, num_pages, eps,
                          q_factors, factor_positions, status};
  auto launch = [&](auto kernel) {
    kernel<<<dim3(tokens, heads + 2 * kv_heads), 256, head_dim * sizeof(float), stream>>>(args);
    return static_cast<int>(cudaGetLastError());
  };
  if (dtype == kF32)
    return kind == kCodesInt8 ? launch(store_quantized_kernel<float, kCodesInt8>) : launch(store_quantized_kernel<float, kCodesE4M3>);
  return kind == kCodesInt8 ? launch(store_quantized_kernel<__nv_bfloat16, kCodesInt8>)
                            : launch(store_quantized_kernel<__nv_bfloat16, kCodesE4M3>);
}

// For each i < rows: the pages of row row_request[i] of the block tables that a
// query at position first[i] or later sees (window, chunk, keep as in the
// attention kernels), up to position last[i], from the pool into `out`, which
// has the pool's layout [pages, 2, kv_heads, page_tokens, head_dim] in `dtype`.
MXB_API int mxb_read_cache(const void* codes, const float* scales, int kind, void* out, int dtype, const int* block_tables, int max_pages,
                           const int* row_request, const int* first, const int* last, int rows, int kv_heads, int head_dim,
                           int page_tokens, int num_pages, int window, int chunk, int keep, int* status, cudaStream_t stream) {
  if (rows <= 0 || max_pages <= 0) return 0;
  if (rows > 65535 || !pool_fits(num_pages, kv_heads, page_tokens) || head_dim <= 0 || head_dim > 512 ||
      (dtype != kF32 && dtype != kBF16) || (kind != kCodesE4M3 && kind != kCodesInt8))
    return static_cast<int>(cudaErrorInvalidValue);
  auto launch = [&](auto kernel, auto* target) {
    kernel<<<dim3(max_pages, rows), 256, 0, stream>>>(static_cast<const uint8_t*>(codes), scales, target, block_tables, max_pages,
                                                     row_request, first, last, kv_heads, head_dim, page_tokens, num_pages, window,
                                                     chunk, keep, status);
    return static_cast<int>(cudaGetLastError());
  };
  if (dtype == kF32)
    return kind == kCodesInt8 ? launch(read_cache_kernel<float, kCodesInt8>, static_cast<float*>(out))
                              : launch(read_cache_kernel<float, kCodesE4M3>, static_cast<float*>(out));
  return kind == kCodesInt8 ? launch(read_cache_kernel<__nv_bfloat16, kCodesInt8>, static_cast<__nv_bfloat16*>(out))
                            : launch(read_cache_kernel<__nv_bfloat16, kCodesE4M3>, static_cast<__nv_bfloat16*>(out));
}
