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

// The same for heads of 64, 128 and 256 values with rotations of whole eights of
// pairs: a lane holds two runs of eight values that contain their own rotation
// partners, HD / 16 lanes make up a head, and sums and maxima run over a head's
// lanes. Run A of lane s starts at 8 s and run B half the rotated values
// further (rotations of halves), or they are neighbours (neighbouring pairs, and
// the values behind the rotated ones); either way the lane needs the cosines
// 8 s ... 8 s + 7. Issue slots and the wait for positions, cosines and rows bind
// it, so warps of queries end at their rotation (2,048 tokens of 32 / 8 heads of
// 128: 20.6 us when they took the codes' part too, 17.6; the write of the same
// rows in bfloat16 takes 14.5). Two or four heads a lane with one set of weights
// and cosines, as that write does it, lose more warps than they save loads
// (20.5 and 22.4 us).
template <typename T, int KIND, int HD>
__global__ void __launch_bounds__(256) store_quantized_lanes_kernel(const __grid_constant__ StoreArgs a) {
  constexpr int LANES = HD / 16, HEADS = 32 / LANES;   // lanes of a head, heads of a warp
  constexpr int WORDS = 8 * sizeof(T) / 16;            // 16-byte words of a run
  chain_release();
  // Up to chain_wait(): only the step's integers and what no kernel of a step writes.
  const int lane = threadIdx.x & 31, sub = lane % LANES;
  const unsigned per_token = a.heads + 2 * a.kv_heads;
  const unsigned total = static_cast<unsigned>(a.tokens) * per_token;   // below 2^31: the launcher sees to it
  const unsigned item = (blockIdx.x * 8u + (threadIdx.x >> 5)) * HEADS + lane / LANES;
  bool active = item < total;   // lanes without work stay to the end: the others exchange values with their warp
  const int t = active ? static_cast<int>(item / per_token) : 0;
  const int h = active ? static_cast<int>(item - static_cast<unsigned>(t) * per_token) : 0;
  const bool is_q = h < a.heads, is_k = !is_q && h < a.heads + a.kv_heads;
  const int kv = is_q ? 0 : (is_k ? h - a.heads : h - a.heads - a.kv_heads);
  const T* src = is_q   ? static_cast<const T*>(a.q_in) + t * a.q_stride + static_cast<long long>(h) * HD
                 : is_k ? static_cast<const T*>(a.k_in) + t * a.k_stride + static_cast<long long>(kv) * HD
                        : static_cast<const T*>(a.v_in) + t * a.v_stride + static_cast<long long>(kv) * HD;
  size_t pool_row = 0;
  if (is_q) {
    if (a.q_out == nullptr) active = false;
  } else if (active) {
    const int slot = a.slots[t], page = slot / a.page_tokens;
    if (slot < 0) {
      active = false;
    } else if (page >= a.num_pages) {
      if (sub == 0) atomicOr(a.status, kStatusBadSlot);
      active = false;
    } else {
      pool_row = ((static_cast<size_t>(page) * 2 + (is_k ? 0 : 1)) * a.kv_heads + kv) * a.page_tokens + (slot - page * a.page_tokens);
    }
  }
  const bool worked = is_q || is_k;   // values are stored as projected
  const int half = a.rotary_dim >> 1;
  const bool rotates = a.cos_table != nullptr, turns = rotates && worked && 16 * sub < a.rotary_dim;
  // runs of halves, where the lane's values are rotated so; else neighbours
  const bool apart = rotates && !a.interleaved && 16 * sub < a.rotary_dim;
  const int at_a = apart ? 8 * sub : 16 * sub, at_b = apart ? half + 8 * sub : 16 * sub + 8;
  const float* weight = is_q ? a.q_weight : (is_k ? a.k_weight : nullptr);
  float gain[16], c[8], sn[8];
  auto floats = [](float* to, const float* from) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float4 x = reinterpret_cast<const float4*>(from)[w];
      to[4 * w] = x.x; to[4 * w + 1] = x.y; to[4 * w + 2] = x.z; to[4 * w + 3] = x.w;
    }
  };
  const bool normed = active && weight != nullptr;
  if (normed) {
    if (a.row_sums != nullptr) weight += static_cast<size_t>(is_q ? h : kv) * HD;   // a norm over the whole projection has weights for every head
    floats(gain, weight + at_a);
    floats(gain + 8, weight + at_b);
  }
  float factor = 1.0f;
  if (active && worked && (rotates || a.q_factors != nullptr)) {
    const int pos = a.positions[t];
    bool there = true;
    if (rotates) there = pos >= 0 && pos < a.table_positions;
    if (turns) {
      const size_t row = static_cast<size_t>(there ? pos : 0) * half + 8 * sub;
      floats(c, a.cos_table + row);
      floats(sn, a.sin_table + row);
    }
    if (is_q && a.q_factors != nullptr) {
      const bool known = pos >= 0 && pos < a.factor_positions;
      factor = a.q_factors[known ? pos : 0];
      there = there && known;
    }
    if (!there && sub == 0) atomicOr(a.status, kStatusBadSlot);
  }
  chain_wait();
  src = behind_wait(src);   // written by the kernel ahead of this one
  alignas(16) T in[16] = {};
  if (active) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      reinterpret_cast<uint4*>(in)[w] = reinterpret_cast<const uint4*>(src + at_a)[w];
      reinterpret_cast<uint4*>(in)[WORDS + w] = reinterpret_cast<const uint4*>(src + at_b)[w];
    }
  }
  float x[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = to_float(in[j]);
  if (a.q_weight != nullptr || a.k_weight != nullptr) {   // the same for the whole launch
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) sum += x[j] * x[j];
#pragma unroll
    for (int offset = LANES / 2; offset > 0; offset >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
    if (normed) {
      const float mean = a.row_sums != nullptr ? behind_wait(a.row_sums)[2 * t + (is_k ? 1 : 0)] : sum / static_cast<float>(HD);
      const float scale = rsqrtf(mean + a.eps);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = x[j] * scale * gain[j];
    }
  }
  if (turns && active) {
    if (a.interleaved) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float lo = x[2 * j], hi = x[2 * j + 1];
        x[2 * j] = lo * c[j] - hi * sn[j];
        x[2 * j + 1] = hi * c[j] + lo * sn[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float lo = x[j], hi = x[8 + j];
        x[j] = lo * c[j] - hi * sn[j];
        x[8 + j] = hi * c[j] + lo * sn[j];
      }
    }
  }
  if (active && is_q) {
    alignas(16) T out[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) out[j] = from_float<T>(x[j] * factor);
    T* dst = static_cast<T*>(a.q_out) + (static_cast<size_t>(t) * a.heads + h) * HD;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      reinterpret_cast<uint4*>(dst + at_a)[w] = reinterpret_cast<const uint4*>(out)[w];
      reinterpret_cast<uint4*>(dst + at_b)[w] = reinterpret_cast<const uint4*>(out)[WORDS + w];
    }
  }
  if (!__any_sync(0xffffffffu, active && !is_q)) return;   // a warp of queries
  float largest = x[0];
#pragma unroll
  for (int j = 1; j < 16; ++j) largest = larger_magnitude(largest, x[j]);
#pragma unroll
  for (int offset = LANES / 2; offset > 0; offset >>= 1)
    largest = larger_magnitude(largest, __shfl_xor_sync(0xffffffffu, largest, offset));
  if (active && !is_q) {
    const RowScale row = row_scale<KIND>(__float_as_uint(largest));
    uint8_t* dst = a.codes + pool_row * HD;
    *reinterpret_cast<uint2*>(dst + at_a) = make_uint2(four_codes<KIND>(x, row), four_codes<KIND>(x + 4, row));
    *reinterpret_cast<uint2*>(dst + at_b) = make_uint2(four_codes<KIND>(x + 8, row), four_codes<KIND>(x + 12, row));
    if (sub == 0) a.scales[pool_row] = row.scale;
  }
}

// Sixteen codes as values of T: exact as halves, times the scale in float32.
__device__ __forceinline__ void store_pair(float* out, float2 v) { *reinterpret_cast<float2*>(out) = v; }
__device__ __forceinline__ void store_pair(__nv_bfloat16* out, float2 v) {
  *reinterpret_cast<__nv_bfloat162*>(out) = __floats2bfloat162_rn(v.x, v.y);
}
template <typename T, int KIND> __device__ __forceinline__ void code_values(const uint4& word, float scale, T* out) {
  const uint32_t words[4] = {word.x, word.y, word.z, word.w};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t halves[2];
    code_halves<KIND>(words[w], halves[0], halves[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&halves[h]));
      store_pair(out + 4 * w + 2 * h, make_float2(v.x * scale, v.y * scale));
    }
  }
}

struct ReadArgs {
  const uint8_t* codes;
  const float* scales;
  void* out;
  const int* block_tables;
  int max_pages;
  const int *row_request, *first, *last;
  int kv_heads, head_dim, page_tokens, num_pages, window, chunk, keep;
  int* status;
};

// Pages back into the compute type, for rows of whole 16-byte pieces: a page's
// codes are one run of memory, and so are its values, so a block takes
// kReadPieces pieces of one page at a time, each thread all its loads in flight
// before the first store. Block (x, request) takes the items x, x + gridDim.x, ...
// of the request's walk over the pages that are seen.
constexpr int kReadThreads = 256, kReadDepth = 2, kReadPieces = kReadThreads * kReadDepth;
constexpr int kReadBlocks = 8 * 148 * 8;   // of a launch, at most (or one a request): eight rounds of what is resident

template <typename T, int KIND>
__global__ void __launch_bounds__(kReadThreads)
read_cache_pieces_kernel(const __grid_constant__ ReadArgs a) {
  // No release ahead of the end: what follows has nothing to do before `out` is there.
  chain_wait();   // the codes are the work of kernels ahead
  // A last position beyond the table is cut to the first one there, whose page is found missing and reported.
  const int end = static_cast<int>(min(static_cast<long long>(a.last[blockIdx.y]), static_cast<long long>(a.max_pages) * a.page_tokens));
  const int row = blockIdx.y, head_dim = a.head_dim, page_tokens = a.page_tokens;
  if (end < 0) return;
  const KeyWalk walk = key_walk(min(first_visible_key(max(a.first[row], 0), a.window, a.chunk), end), end, a.keep, page_tokens);
  const int per_row = head_dim >> 4, rows = 2 * a.kv_heads * page_tokens, pieces = rows * per_row;
  const int per_page = (pieces + kReadPieces - 1) / kReadPieces;
  const int* table = a.block_tables + static_cast<size_t>(a.row_request[row]) * a.max_pages;
  for (int item = blockIdx.x; item < walk.count * per_page; item += gridDim.x) {
    const int step = item / per_page, slot = walk.tile(step), piece0 = (item - step * per_page) * kReadPieces;
    const int page = slot < a.max_pages ? table[slot] : -1;
    if (page < 0 || page >= a.num_pages) {
      if (threadIdx.x == 0) atomicOr(a.status, kStatusBadPage);
      continue;
    }
    const int seen = end - slot * page_tokens + 1;   // rows of the page up to the last position
    const size_t base = static_cast<size_t>(page) * rows;
    const uint4* src = reinterpret_cast<const uint4*>(a.codes + base * head_dim);
    uint4 held[kReadDepth];
    float scale[kReadDepth];
    bool there[kReadDepth];
#pragma unroll
    for (int j = 0; j < kReadDepth; ++j) {
      const int piece = piece0 + j * kReadThreads + threadIdx.x, line = piece / per_row;
      there[j] = piece < pieces && (seen >= page_tokens || line % page_tokens < seen);
      held[j] = there[j] ? src[piece] : make_uint4(0u, 0u, 0u, 0u);
      scale[j] = there[j] ? a.scales[base + line] : 0.0f;
    }
    T* dst = static_cast<T*>(a.out) + base * head_dim;
#pragma unroll
    for (int j = 0; j < kReadDepth; ++j) {
      if (!there[j]) continue;
      alignas(16) T values[16];
      code_values<T, KIND>(held[j], scale[j], values);
      uint4* to = reinterpret_cast<uint4*>(dst + static_cast<size_t>(piece0 + j * kReadThreads + threadIdx.x) * 16);
#pragma unroll
      for (int w = 0; w < static_cast<int>(sizeof(T)); ++w) to[w] = reinterpret_cast<const uint4*>(values)[w];
    }
  }
}

// The general form, a code at a time: block (page of the table, request). The
// rows up to the request's last position are written, everything else of
// `out` stays as it is.
template <typename T, int KIND>
__global__ void __launch_bounds__(256)
read_cache_kernel(const __grid_constant__ ReadArgs a) {
  chain_wait();
  const int slot = blockIdx.x, row = blockIdx.y;
  const int begin = first_visible_key(max(a.first[row], 0), a.window, a.chunk), end = a.last[row];
  if (end < 0) return;
  const int last_slot = end / a.page_tokens;
  if (slot == 0 && last_slot >= a.max_pages && threadIdx.x == 0) atomicOr(a.status, kStatusBadPage);   // `last` lies beyond the table
  if (slot > last_slot || slot >= a.max_pages) return;
  const int key0 = slot * a.page_tokens;
  if (key0 + a.page_tokens <= begin && key0 >= a.keep) return;
  const int page = a.block_tables[static_cast<size_t>(a.row_request[row]) * a.max_pages + slot];
  if (page < 0 || page >= a.num_pages) {
    if (threadIdx.x == 0) atomicOr(a.status, kStatusBadPage);
    return;
  }
  const int rows = min(end - key0, a.page_tokens - 1) + 1;
  const size_t base = static_cast<size_t>(page) * 2 * a.kv_heads * a.page_tokens;
  for (int i = threadIdx.x; i < 2 * a.kv_heads * rows * a.head_dim; i += blockDim.x) {
    const int line = i / a.head_dim, d = i - line * a.head_dim;
    const int head = line / rows, r = line - head * rows;
    const size_t at = base + static_cast<size_t>(head) * a.page_tokens + r;
    static_cast<T*>(a.out)[at * a.head_dim + d] = from_float<T>(code_value<KIND>(a.codes[at * a.head_dim + d]) * a.scales[at]);
  }
}

}  // namespace mxb

using namespace mxb;

static bool pool_fits(int num_pages, int kv_heads, int page_tokens) {
  return num_pages > 0 && kv_heads > 0 && page_tokens > 0 &&
         static_cast<long long>(num_pages) * 2 * kv_heads * page_tokens <= 0x7fffffffLL;
}

// What mxb_store_quantized is asked for, 8 bytes a field.
struct StoreCall {
  const void *q_in, *k_in, *v_in;
  void *q_out, *codes;
  float* scales;
  const int *slots, *positions;
  const float *q_weight, *k_weight, *cos_table, *sin_table;
  float* row_sums;
  const float* q_factors;
  int* status;
  long long q_stride, k_stride, v_stride, kind, dtype, table_positions, rotary_dim, interleaved, norm_scope, tokens, heads, kv_heads,
      head_dim, page_tokens, num_pages, factor_positions;
  double eps;
};

// The norm and rotation of a step's queries and keys, queries to q_out, keys and
// values into the pool as codes at `slots` (negative: not written). row_sums:
// float32 scratch of 2 * tokens values for norm_scope 1 (a norm over a token's
// whole projection; weights [heads * head_dim] and [kv_heads * head_dim]).
MXB_API int mxb_store_quantized(const void* call, int bytes, cudaStream_t stream) {
  if (bytes != static_cast<int>(sizeof(StoreCall))) return static_cast<int>(cudaErrorInvalidValue);
  const StoreCall& c = *static_cast<const StoreCall*>(call);
  if (c.tokens <= 0) return 0;
  const int kind = static_cast<int>(c.kind), dtype = static_cast<int>(c.dtype), tokens = static_cast<int>(c.tokens),
            heads = static_cast<int>(c.heads), kv_heads = static_cast<int>(c.kv_heads), head_dim = static_cast<int>(c.head_dim),
            page_tokens = static_cast<int>(c.page_tokens), num_pages = static_cast<int>(c.num_pages);
  if (c.codes == nullptr || c.scales == nullptr || c.slots == nullptr || !pool_fits(num_pages, kv_heads, page_tokens) || head_dim <= 0 ||
      head_dim > 512 || heads < 0 || heads + 2 * kv_heads > 65535 || c.rotary_dim < 0 || c.rotary_dim > head_dim || (c.rotary_dim & 1) ||
      (dtype != kF32 && dtype != kBF16) || (kind != kCodesE4M3 && kind != kCodesInt8) || (c.norm_scope == 1 && c.row_sums == nullptr))
    return static_cast<int>(cudaErrorInvalidValue);
  if (c.norm_scope == 1 && (c.q_weight != nullptr || c.k_weight != nullptr)) {
    const dim3 grid(tokens, 2);
    if (dtype == kF32)
      projection_squares_kernel<float><<<grid, 256, 0, stream>>>(static_cast<const float*>(c.q_in), static_cast<const float*>(c.k_in), c.q_stride,
                                                                  c.k_stride, heads * head_dim, kv_heads * head_dim, c.row_sums);
    else
      projection_squares_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(
          static_cast<const __nv_bfloat16*>(c.q_in), static_cast<const __nv_bfloat16*>(c.k_in), c.q_stride, c.k_stride,
          heads * head_dim, kv_heads * head_dim, c.row_sums);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  const StoreArgs args = {c.q_in, c.k_in, c.v_in, c.q_stride, c.k_stride, c.v_stride, c.q_out, static_cast<uint8_t*>(c.codes), c.scales,
                          c.slots, c.positions, c.q_weight, c.k_weight, c.cos_table, c.sin_table, static_cast<int>(c.table_positions),
                          static_cast<int>(c.rotary_dim), static_cast<int>(c.interleaved), c.norm_scope == 1 ? c.row_sums : nullptr,
                          tokens, heads, kv_heads, head_dim, page_tokens, num_pages, static_cast<float>(c.eps), c.q_factors,
                          static_cast<int>(c.factor_positions), c.status};
  // The lanes' form: 16-byte accesses throughout, runs of eight that hold their rotation partners.
  const int element = dtype == kF32 ? 4 : 2;
  auto aligned = [&](const void* p, long long stride) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * element) % 16 == 0);
  };
  const long long items = static_cast<long long>(tokens) * (heads + 2 * kv_heads);
  if ((head_dim == 64 || head_dim == 128 || head_dim == 256) && items < 0x7fffffffLL && c.rotary_dim % 16 == 0 &&
      aligned(c.q_in, c.q_stride) && aligned(c.k_in, c.k_stride) && aligned(c.v_in, c.v_stride) && aligned(c.q_out, 0) &&
      aligned(c.codes, 0) && aligned(c.q_weight, 0) && aligned(c.k_weight, 0) && aligned(c.cos_table, 0) && aligned(c.sin_table, 0)) {
    const int heads_per_block = 8 * (32 / (head_dim / 16));
    const dim3 grid(static_cast<unsigned>((items + heads_per_block - 1) / heads_per_block));
    auto launch = [&](auto kernel) { return static_cast<int>(launch_chained(kernel, grid, dim3(256), 0, stream, args)); };
#define BY_SIZE(T, KIND) (head_dim == 64    ? launch(store_quantized_lanes_kernel<T, KIND, 64>)  \
                          : head_dim == 128 ? launch(store_quantized_lanes_kernel<T, KIND, 128>) \
                                            : launch(store_quantized_lanes_kernel<T, KIND, 256>))
    if (dtype == kF32) return kind == kCodesInt8 ? BY_SIZE(float, kCodesInt8) : BY_SIZE(float, kCodesE4M3);
    return kind == kCodesInt8 ? BY_SIZE(__nv_bfloat16, kCodesInt8) : BY_SIZE(__nv_bfloat16, kCodesE4M3);
#undef BY_SIZE
  }
  auto launch = [&](auto kernel) {
    kernel<<<dim3(tokens, heads + 2 * kv_heads), 256, head_dim * sizeof(float), stream>>>(args);
    return static_cast<int>(cudaGetLastError());
  };
  if (dtype == kF32)
    return kind == kCodesInt8 ? launch(store_quantized_kernel<float, kCodesInt8>) : launch(store_quantized_kernel<float, kCodesE4M3>);
  return kind == kCodesInt8 ? launch(store_quantized_kernel<__nv_bfloat16, kCodesInt8>)
                            : launch(store_quantized_kernel<__nv_bfloat16, kCodesE4M3>);
}

// What mxb_read_cache is asked for, 8 bytes a field.
struct ReadCall {
  const void* codes;
  const float* scales;
  void* out;
  const int *block_tables, *row_request, *first, *last;
  int* status;
  long long kind, dtype, max_pages, rows, kv_heads, head_dim, page_tokens, num_pages, window, chunk, keep;
};

// For each i < rows: the pages of row row_request[i] of the block tables that a
// query at position first[i] or later sees (window, chunk, keep as in the
// attention kernels), up to position last[i], from the pool into `out`, which
// has the pool's layout [pages, 2, kv_heads, page_tokens, head_dim] in `dtype`.
// Positions beyond the table are reported (a bad page); what the table has of them is read.
MXB_API int mxb_read_cache(const void* call, int bytes, cudaStream_t stream) {
  if (bytes != static_cast<int>(sizeof(ReadCall))) return static_cast<int>(cudaErrorInvalidValue);
  const ReadCall& c = *static_cast<const ReadCall*>(call);
  if (c.rows <= 0) return 0;
  const int kind = static_cast<int>(c.kind), dtype = static_cast<int>(c.dtype), rows = static_cast<int>(c.rows),
            kv_heads = static_cast<int>(c.kv_heads), head_dim = static_cast<int>(c.head_dim), max_pages = static_cast<int>(c.max_pages),
            page_tokens = static_cast<int>(c.page_tokens), num_pages = static_cast<int>(c.num_pages);
  if (rows > 65535 || max_pages < 0 || !pool_fits(num_pages, kv_heads, page_tokens) || head_dim <= 0 || head_dim > 512 ||
      2LL * kv_heads * page_tokens * head_dim > 0x7fffffffLL ||   // a page's codes are counted in 31 bits
      (dtype != kF32 && dtype != kBF16) || (kind != kCodesE4M3 && kind != kCodesInt8))
    return static_cast<int>(cudaErrorInvalidValue);
  const bool by_pieces = head_dim % 16 == 0 && reinterpret_cast<uintptr_t>(c.codes) % 16 == 0 && reinterpret_cast<uintptr_t>(c.out) % 16 == 0;
  // A block an item where tables are short; wide tables of short contexts (a captured step's) walk with a stride instead.
  const long long items = static_cast<long long>(max_pages) * ((2LL * kv_heads * page_tokens * (head_dim / 16) + kReadPieces - 1) / kReadPieces);
  const long long most = kReadBlocks / rows > 0 ? kReadBlocks / rows : 1;
  const long long blocks = !by_pieces ? max_pages : (items < most ? items : most);
  const dim3 grid(static_cast<unsigned>(blocks > 0 ? blocks : 1), rows);   // a table without pages: a block that says so
  const ReadArgs args = {static_cast<const uint8_t*>(c.codes), c.scales, c.out, c.block_tables, max_pages, c.row_request, c.first, c.last,
                         kv_heads, head_dim, page_tokens, num_pages, static_cast<int>(c.window), static_cast<int>(c.chunk),
                         static_cast<int>(c.keep), c.status};
  auto launch = [&](auto kernel) { return static_cast<int>(launch_chained(kernel, grid, dim3(kReadThreads), 0, stream, args)); };
#define BY_TYPE(KERNEL) (dtype == kF32 ? (kind == kCodesInt8 ? launch(KERNEL<float, kCodesInt8>) : launch(KERNEL<float, kCodesE4M3>)) \
                                       : (kind == kCodesInt8 ? launch(KERNEL<__nv_bfloat16, kCodesInt8>) : launch(KERNEL<__nv_bfloat16, kCodesE4M3>)))
  return by_pieces ? BY_TYPE(read_cache_pieces_kernel) : BY_TYPE(read_cache_kernel);
#undef BY_TYPE
}

MXB_TIMELINE_EXPORT(mxb_timeline_quantized_cache)
