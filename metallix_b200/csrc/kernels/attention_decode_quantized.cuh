// Attention of single decoded tokens over a cache held in 8 bits (the rows of
// quantized.cuh): scores s_j = (q . code_j) scale_j, softmax, and the sum of
// (p_j scale_j) code_j, in float32, without ever making the rows themselves.
//
// Work is cut as the kernels over a cache in the compute type cut it: a pair of
// (token, key/value head) gets `slots` blocks, block s takes the tiles of
// kSplitKeys keys first + s, first + s + slots, ... of the token's keys and ends with
// one unnormalised partial result (accumulator, maximum, sum). Those of a pair are
// put together in slot order, by the merge kernel or, where a pair's blocks are
// few enough to be one cluster, by the blocks themselves out of one another's
// shared memory.
#pragma once

#include "quantized.cuh"

namespace mxb {

struct QuantizedDecode {
  const void* q;                 // [tokens, heads, head_dim]
  const uint8_t* codes;
  const float* scales;
  float* partial;                // [rows, heads, slots, head_dim + 2]
  const int* block_tables;
  int max_pages, table_rows;     // what the block tables have of columns and rows
  const int *row_token, *row_request, *positions;
  int heads, kv_heads, head_dim, page_tokens, num_pages, window, chunk, keep;
  float scale, softcap;
  ScoreBias bias;
  int group;                     // query heads a key/value head
  int page_shift;                // log2 of page_tokens, -1 where that is no power of two
  int settled;                   // the positions ahead of each token's own were complete when the launch ahead of this one began
  int* status;
  // What the blocks of a cluster write where they put their results together themselves (`fused`: the slots of a pair are one cluster).
  int fused, max_splits;
  void* out;                     // [tokens, heads, head_dim]
  const void* gate;              // optional, rows gate_stride values apart
  long long gate_stride;
  int has_sink;
  float sink_score;
  const float* sink_heads;
};

constexpr int kQuantHeads = 8;   // query heads of a block of the general kernel

// The general form: every head size up to 256 and any number of query heads a
// key/value head. A warp takes a key at a time, a lane every 32nd value.
template <typename T, int KIND, int VALUES>
__global__ void __launch_bounds__(kDecodeThreads)
quantized_decode_kernel(const QuantizedDecode a) {
  constexpr int G = kQuantHeads, WARPS = kDecodeThreads / 32;
  __shared__ float s_acc[WARPS][32 * VALUES];
  __shared__ float s_stat[WARPS][G][2];
  const int rank = blockIdx.x, slots = gridDim.x, kv = blockIdx.y % a.kv_heads, part = blockIdx.y / a.kv_heads, row = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int token = a.row_token[row];
  if (token < 0) return;   // a padding row
  const int pos = a.positions[token], group = a.heads / a.kv_heads;
  const int live = min(group - part * G, G), head0 = kv * group + part * G;   // this block's query heads
  const int first_key = first_visible_key(pos, a.window, a.chunk);
  const KeyWalk walk = key_walk(first_key, pos, a.keep, kSplitKeys);
  if (rank >= walk.count) return;   // more slots than tiles: the merge skips this one
  const int* table = a.block_tables + static_cast<size_t>(a.row_request[row]) * a.max_pages;
  const int n = a.head_dim;

  float q[G][VALUES], o[G][VALUES], m[G], l[G];
#pragma unroll
  for (int h = 0; h < G; ++h) {
    m[h] = kDecodeMinusHuge;
    l[h] = 0.0f;
#pragma unroll
    for (int i = 0; i < VALUES; ++i) {
      const int d = lane + 32 * i;
      q[h][i] = h < live && d < n ? to_float(static_cast<const T*>(a.q)[(static_cast<size_t>(token) * a.heads + head0 + h) * n + d]) : 0.0f;
      o[h][i] = 0.0f;
    }
  }
  for (int step = rank; step < walk.count; step += slots) {
    const int key0 = walk.tile(step) * kSplitKeys + warp * 32;
    for (int key = key0; key < key0 + 32 && key <= pos; ++key) {
      if (!key_seen(key, pos, first_key, a.keep)) continue;
      const int at = quantized_row(table, a.max_pages, a.num_pages, a.kv_heads, kv, a.page_tokens, key, a.status);
      if (at < 0) continue;
      const size_t k_row = at, v_row = k_row + static_cast<size_t>(a.kv_heads) * a.page_tokens;
      const float k_scale = a.scales[k_row], v_scale = a.scales[v_row];
      float k[VALUES], v[VALUES];
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        const int d = lane + 32 * i;
        k[i] = d < n ? code_value<KIND>(a.codes[k_row * n + d]) * k_scale : 0.0f;   // q . code may leave float32 where the score does not
        v[i] = d < n ? code_value<KIND>(a.codes[v_row * n + d]) : 0.0f;
      }
#pragma unroll
      for (int h = 0; h < G; ++h) {
        if (h >= live) continue;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) s = fmaf(q[h][i], k[i], s);
        s = capped_score(warp_sum(s) * a.scale, a.softcap);
        if (a.bias.table != nullptr) s += bias_at(a.bias.row(head0 + h), pos - key, a.bias.far);
        const float top = fmaxf(m[h], s), carry = expf(m[h] - top), p = expf(s - top);
        m[h] = top;
        l[h] = fmaf(l[h], carry, p);
#pragma unroll
        for (int i = 0; i < VALUES; ++i) o[h][i] = fmaf(p * v_scale, v[i], o[h][i] * carry);
      }
    }
  }
  // the four warps' results in warp order, head by head
  for (int h = 0; h < G; ++h)
    if (lane == 0) { s_stat[warp][h][0] = m[h]; s_stat[warp][h][1] = l[h]; }
#pragma unroll
  for (int h = 0; h < G; ++h) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VALUES; ++i) s_acc[warp][lane + 32 * i] = o[h][i];
    __syncthreads();
    if (h >= live) continue;
    float top = kDecodeMinusHuge, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_stat[w][h][0]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum = fmaf(s_stat[w][h][1], expf(s_stat[w][h][0] - top), sum);
    float* dst = a.partial + ((static_cast<size_t>(row) * a.heads + head0 + h) * slots + rank) * (n + 2);
    for (int d = threadIdx.x; d < n; d += kDecodeThreads) {
      float value = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) value = fmaf(s_acc[w][d], expf(s_stat[w][h][0] - top), value);
      dst[d] = value;
    }
    if (threadIdx.x == 0) { dst[n] = top; dst[n + 1] = sum; }
  }
}

// ---------------------------------------------------------------------------
// The same on the tensor cores, for heads of 64, 128 and 256 values. Codes of
// either kind are exact in half precision, so the products q . code and p . code
// are mma.sync m16n8k16 of halves with float32 sums, the scales joining behind
// and ahead of them. Long contexts are bound by the codes' bytes only if what is
// done to a code costs next to nothing: a pair of e4m3 codes becomes two halves
// by one conversion (and a shuffle of bytes for every four codes of V), a pair of
// whole numbers by three instructions.
//
// Halves reach from 2^-24 to 2^16, which powers of two make room for: a head's
// queries are scaled so that the largest lies at 2^14 (what is lost below is
// 2^-39 of it), and the weights p_j scale_j by `up`, so that the largest lies at
// 2^kQuantTop when they are first looked at and may grow up to 2^15. The same
// goes for the maximum that the exponentials are taken against: it is found by
// exchanging values only when a stage's sum or weights outgrow their room, so
// that most stages exchange nothing. What a warp has gathered is
//   sum_j 2^(s_j - m) scale_j code_j * up   and   sum_j 2^(s_j - m)
// for any m, which need not be the maximum.
//
// A warp works alone until the end: it takes its 32 keys of a 128-key tile (a
// stage; for heads of 256, 16 of them) and has their rows brought into a ring of
// its own by TMA, one box per page and plane with the swizzle that lets its lanes
// read them without bank conflicts. (With copies of 16 bytes a lane by cp.async
// 8 requests over 32,000 positions took 113 to 130 us, whatever depth and number
// of blocks an SM was tried; by TMA 90.)
// What a lane reads is chosen so that bytes need no transposing:
//   K: lane (g, t) = (lane / 4, lane % 4) reads the 16-byte chunks 2t, 2t + 1 of the
//      key g of eight (heads of 64: chunk t). Word w of a chunk of the keys g and
//      g + 8 is the A operand of one 16-value step (scores^T = K q^T: 16 keys by 8
//      query heads); q's registers follow the same order of values.
//   V: lane (g, t) reads chunk g of the keys 2t, 2t + 1, 2t + 8, 2t + 9, from which
//      byte pairs of neighbouring keys make the A operand (o^T = V^T p^T: 16 values
//      of a row by 8 query heads). p^T's B operand is the scores' tile turned by
//      movmatrix. No row of either product is wasted.
//
// float32 queries are two halves each, 22 bits and the sign of what is left; so
// are the weights: a second product for either. For bfloat16 queries, which one
// half holds whole, the weights are one half, eleven bits, three more than the
// output's; the sum that they are divided by takes them unrounded.
template <int HD> struct QuantTile {
  static constexpr int kKeys = HD == 256 ? 16 : 32;            // of a stage
  static constexpr int kBlocks8 = kKeys / 8;                   // eights of keys
  static constexpr int kChunks = HD / 64;                      // 16-byte chunks of a key row a lane takes
  static constexpr int kValueBytes = HD >= 128 ? 16 : HD / 8;  // of a value row a lane takes at once
  static constexpr int kValuePieces = HD / 8 / kValueBytes;
  static constexpr int kBoxBytes = HD >= 128 ? 128 : HD;       // of a row in one box; heads of 256 lie as two halves
  static constexpr int kRowBytes = kKeys * HD;                 // a stage's keys; its values as many
  static constexpr int kStages = HD == 128 ? 2 : 3;
  static constexpr int kWarpBytes = kStages * 2 * kRowBytes;   // the ring's codes; its scales lie behind all warps' codes
  static constexpr int kScales = 2 * kKeys;                    // of a stage: keys', values'
  static constexpr int kRing = (kDecodeThreads / 32) * (kWarpBytes + kStages * kScales * 4);
  static constexpr int kMerge = (kDecodeThreads / 32 + 1) * 8 * (HD + 2) * 4;   // the warps' results and the block's
  static constexpr int kShared = (kRing > kMerge ? kRing : kMerge) + 1024;   // and room to align to the swizzle's period
  // Where chunk c of row r of a stage lies: the hardware's swizzle of 128-byte rows (64-byte ones for heads of 64).
  static __device__ __forceinline__ int at(int r, int c) {
    return HD == 64 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4) : (c >> 3) * (kKeys * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  }
};

__device__ __forceinline__ void quant_copy_scale(float* dst, const float* src, bool there) {
  const uint32_t address = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(address), "l"(src), "r"(there ? 4 : 0));   // else zero
}

// A pool's codes as [rows, head_dim] bytes, read in boxes of box_rows rows. Encoded anew for every call.
static bool encode_codes_map(CUtensorMap* map, const void* codes, long long rows, int head_dim, int box_rows) {
  EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  const int box = head_dim >= 128 ? 128 : head_dim;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(head_dim)};
  const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(box), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t element_strides[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, boxes, element_strides,
                CU_TENSOR_MAP_INTERLEAVE_NONE, box == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

__device__ __forceinline__ void quant_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kQuantTop = 6;
constexpr float kQuantLow = -1.0e30f;   // the reference before the first key: any score is far above it

// An 8 x 8 tile of halves, two of a row a lane, turned.
__device__ __forceinline__ uint32_t turn_tile(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

// A pair of float32 numbers as PARTS pairs of halves, largest first.
template <int PARTS> __device__ __forceinline__ void split_pair(float x, float y, uint32_t (&out)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const __half2 part = __floats2half2_rn(x, y);
    out[i] = *reinterpret_cast<const uint32_t*>(&part);
    x -= __low2float(part);
    y -= __high2float(part);
  }
}

__device__ __forceinline__ float power_of_two(int exponent) { return __uint_as_float(static_cast<uint32_t>(exponent + 127) << 23); }

template <typename T> __device__ __forceinline__ float quant_exp2(float x) { return std::is_same<T, float>::value ? exp2f(x) : decode_exp2(x); }

__device__ __forceinline__ void quant_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
}
// What lies at `mine` in the shared memory of the cluster's block `rank`.
__device__ __forceinline__ float quant_peer(const float* mine, int rank) {
  uint32_t address;
  float value;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(address) : "r"(shared_address(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(value) : "r"(address) : "memory");
  return value;
}

// Blocks resident on an SM: what the ring and the registers leave room for. Heads of 64 (bfloat16) have room for a fourth,
// which is worth little: 8 requests of 32,000 positions 61 us with three and 58 with four, 61 ragged ones 55 and 55.
template <typename T, int HD> struct QuantBlocks {
  static constexpr int value = HD == 256 ? (std::is_same<T, float>::value ? 1 : 2) : 3;
};

template <typename T, int KIND, int HD, bool BIASED>
__global__ void __launch_bounds__(kDecodeThreads, QuantBlocks<T, HD>::value)
quantized_decode_mma_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ QuantizedDecode a) {
  using Tile = QuantTile<HD>;
  constexpr int PARTS = std::is_same<T, float>::value ? 2 : 1;
  constexpr int WARPS = kDecodeThreads / 32, STAGES = Tile::kStages, STEPS = HD / 16, KEYS = Tile::kKeys, EIGHTS = Tile::kBlocks8;
  constexpr int HALVES = 32 / KEYS;   // stages of a warp's 32 keys of a tile
  constexpr float kLog2E = 1.4426950408889634f;
  extern __shared__ unsigned char quant_raw[];
  __shared__ __align__(8) uint64_t barriers[WARPS * STAGES];
  unsigned char* quant_shared = quant_raw + ((1024 - (shared_address(quant_raw) & 1023)) & 1023);
  const bool release_late = gridDim.x * gridDim.y * gridDim.z > QuantBlocks<T, HD>::value * 148u;   // as in the kernels over bfloat16 rows
  if (!release_late) chain_release();
  const int rank = blockIdx.x, slots = gridDim.x, row = blockIdx.z, group = a.group;
  int kv = blockIdx.y, part = 0;   // key/value head, and which eight of its query heads
  for (; kv >= a.kv_heads; kv -= a.kv_heads) ++part;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  // Pages are a power of two of 8 positions or more: a box is a page's rows of one plane, or of a stage where a page has more.
  // Lane n has box n fetched (keys' boxes, then values'; for heads of 256 each as two halves) and looks after key n's scales.
  // Pages are asked for one stage ahead of the copies, and looked at only then; those of the first stage together with the
  // position, on the guess that neither a window nor a chunk has moved the first tile.
  constexpr int WIDE = HD / Tile::kBoxBytes, KEYS_LOG = KEYS == 32 ? 5 : 4, WIDE_LOG = WIDE - 1;   // WIDE boxes a row is cut into: 1 or 2
  const int shift = a.page_shift, in_page = a.page_tokens - 1, box_shift = min(shift, KEYS_LOG), box_keys = 1 << box_shift;
  const int plane_log = KEYS_LOG - box_shift + WIDE_LOG, boxes = 2 << plane_log;   // boxes of a plane, as a power of two
  const int plane = lane >> plane_log, box = (lane & ((1 << plane_log) - 1)) >> WIDE_LOG, wide = lane & (WIDE - 1);
  const int box_key = box << box_shift, scale_key = lane % KEYS;
  if (!a.settled) chain_wait();
  const int token = a.row_token[row], request = a.row_request[row];
  uint64_t* landed = barriers + warp * STAGES;
  if (lane == 0) {   // while those are on their way
#pragma unroll
    for (int i = 0; i < STAGES; ++i) barrier_init(&landed[i], 1);
    barrier_init_fence();
  }
  __syncwarp();
  auto guess_at = [&](int key) {   // a padding row's request may be no row of the tables
    return (key >> shift) < a.max_pages ? a.block_tables[table_entry(request, key >> shift, a.max_pages, a.table_rows)] : -1;
  };
  int box_page = guess_at(rank * kSplitKeys + warp * 32 + box_key), scale_page = guess_at(rank * kSplitKeys + warp * 32 + scale_key);
  if (token < 0) {
    chain_wait();   // a launch that ends ahead of the one before it lets what follows start too early
    return;
  }
  const int* table = a.block_tables + static_cast<size_t>(request) * a.max_pages;
  auto page_at = [&](int key) { return (key >> shift) < a.max_pages ? table[key >> shift] : -1; };
  const int pos = a.positions[token];
  const int live = min(group - part * 8, 8), head0 = kv * group + part * 8;   // this block's query heads
  const int first_key = first_visible_key(pos, a.window, a.chunk);
  const KeyWalk walk = key_walk(first_key, pos, a.keep, kSplitKeys);
  if (pos / kSplitKeys >= a.max_splits) {   // beyond the caller's bound on the contexts: the row is left as it is
    if (a.fused && rank == 0 && threadIdx.x == 0) atomicOr(a.status, kStatusBadSlot);
    chain_wait();
    return;
  }
  // The end of a pair whose blocks are a cluster: every block's partial result lies at `results` in its shared memory,
  // [8 heads][HD + 2] with maxima in powers of two, and a block writes every slots-th part of the output.
  float* results = reinterpret_cast<float*>(quant_shared) + WARPS * 8 * (HD + 2);
  auto finish = [&]() {
    if (slots > 1) quant_cluster_sync();
    else __syncthreads();
    const int parts_in = min(slots, walk.count);   // the others have nothing
    for (int i = rank * kDecodeThreads + threadIdx.x; i < live * HD; i += slots * kDecodeThreads) {
      const int h = i / HD, d = i - h * HD;
      float m_all = kQuantLow, sum = 0.0f, l_all = 0.0f;
      for (int b = 0; b < parts_in; ++b) m_all = fmaxf(m_all, quant_peer(results + h * (HD + 2) + HD, b));
      for (int b = 0; b < parts_in; ++b) {
        const float weight = quant_exp2<T>(quant_peer(results + h * (HD + 2) + HD, b) - m_all);
        sum = fmaf(weight, quant_peer(results + h * (HD + 2) + d, b), sum);
        l_all = fmaf(weight, quant_peer(results + h * (HD + 2) + HD + 1, b), l_all);
      }
      const int head = head0 + h;
      if (a.has_sink) l_all += quant_exp2<T>((a.sink_heads != nullptr ? a.sink_heads[head] : a.sink_score) * kLog2E - m_all);
      float value = sum / l_all;
      if (a.gate != nullptr) {
        const T* gate = behind_wait(static_cast<const T*>(a.gate)) + token * a.gate_stride;
        value *= sigmoid_of(to_float(gate[static_cast<long long>(head) * HD + d]));
      }
      static_cast<T*>(a.out)[(static_cast<size_t>(token) * a.heads + head) * HD + d] = from_float<T>(value);
    }
    if (slots > 1) quant_cluster_sync();   // nobody leaves while its results are being read
  };
  if (rank >= walk.count) {   // more slots than tiles
    if (a.fused) {
      chain_wait();
      finish();
    }
    return;
  }
  unsigned char* ring = quant_shared + warp * Tile::kWarpBytes;
  float* ring_scales = reinterpret_cast<float*>(quant_shared + WARPS * Tile::kWarpBytes) + warp * (STAGES * Tile::kScales);

  // Stage i of the warp: part i % HALVES of its keys of the block's tile i / HALVES.
  const int stages = HALVES * ((walk.count - rank + slots - 1) / slots);
  auto first_of = [&](int i) { return walk.tile(rank + i / HALVES * slots) * kSplitKeys + warp * 32 + i % HALVES * KEYS; };
  auto holds = [&](int key0) { return key0 <= pos && (key0 + KEYS > first_key || key0 < a.keep); };
  auto wanted = [&](int key, int keys) { return key <= pos && (key + keys > first_key || key < a.keep); };
  auto page_of = [&](int i, int key) { return i < stages ? page_at(first_of(i) + key) : -1; };   // of key `key` of stage i
  const int value_rows = a.kv_heads * a.page_tokens;   // from a key's row to its value's
  auto row_in = [&](int page, int key) { return (page * 2 * a.kv_heads + kv) * a.page_tokens + (key & in_page); };
  // Every box of a stage is fetched: one that holds nothing the token sees starts behind the pool's last row, where the
  // copy engine finds zeros.
  auto issue = [&](int i, int box_page, int scale_page) {
    if (i < stages) {
      const int slot = i % STAGES, key0 = first_of(i);
      if (lane == 0) barrier_arrive_expect(&landed[slot], 2 * Tile::kRowBytes);
      __syncwarp();
      if (lane < boxes) {
        const int key = key0 + box_key;
        bool there = wanted(key, box_keys);
        if (there && (box_page < 0 || box_page >= a.num_pages)) {
          atomicOr(a.status, kStatusBadPage);
          there = false;
        }
        tma_load_2d(ring + slot * (2 * Tile::kRowBytes) + plane * Tile::kRowBytes + wide * (KEYS * 128) + box_key * Tile::kBoxBytes,
                    &map_codes, wide * Tile::kBoxBytes,
                    there ? row_in(box_page, key) + plane * value_rows : a.num_pages * 2 * value_rows, &landed[slot]);
      }
      const int key = key0 + lane % KEYS;
      const bool there = key_seen(key, pos, first_key, a.keep) && scale_page >= 0 && scale_page < a.num_pages;
      const float* scale = a.scales + (there ? row_in(scale_page, key) : 0);
      float* to = ring_scales + slot * Tile::kScales + lane;
      if (KEYS == 32) {
        quant_copy_scale(to, scale, there);
        quant_copy_scale(to + KEYS, scale + value_rows, there);
      } else {
        quant_copy_scale(to, scale + (lane < KEYS ? 0 : value_rows), there);
      }
    }
    asm volatile("cp.async.commit_group;\n" ::);
  };
  // The token's own row, of the walk's last tile, is written by the kernel ahead of this one; with `settled` all others
  // were complete when that kernel began, and their copies start ahead of the wait.
  bool waited = !a.settled;
  if (walk.tile(rank) != rank) {
    box_page = page_of(0, box_key);
    scale_page = page_of(0, scale_key);
  }
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (!waited && i < stages && first_of(i) + KEYS > pos) {
      chain_wait();
      waited = true;
    }
    const int next_box = page_of(i + 1, box_key), next_scale = page_of(i + 1, scale_key);
    issue(i, box_page, scale_page);
    box_page = next_box;
    scale_page = next_scale;
  }
  if (!waited) chain_wait();

  // ---- the query heads as rows 0..7 (float32: their second halves as rows 8..15)
  auto key_chunk = [&](int j) { return HD == 64 ? t : (j >> 1) * 8 + 2 * t + (j & 1); };   // the lane's j-th chunk of a key row
  const bool scaled = BIASED || a.softcap > 0.0f;   // scores in natural units first; else in powers of two at once
  uint32_t q0[STEPS][PARTS], q2[STEPS][PARTS];
  float score_scale;
  {
    const T* q = behind_wait(static_cast<const T*>(a.q)) + (static_cast<size_t>(token) * a.heads + head0 + (g < live ? g : 0)) * HD;
    alignas(16) T values[STEPS][4];
    uint32_t largest = 0;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const T* at = q + key_chunk(s >> 2) * 16 + (s & 3) * 4;
      if (PARTS == 1) *reinterpret_cast<uint2*>(values[s]) = *reinterpret_cast<const uint2*>(at);
      else *reinterpret_cast<uint4*>(values[s]) = *reinterpret_cast<const uint4*>(at);
#pragma unroll
      for (int i = 0; i < 4; ++i) largest = max(largest, magnitude_bits(to_float(values[s][i])));
    }
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
    // a head that is not finite shows it in its scores whatever the power
    const int up = largest >= 0x7f800000u ? 0 : min(14 + 127 - static_cast<int>(largest >> 23), 126);
    const float power = g < live ? power_of_two(up) : 0.0f;
    score_scale = a.scale * power_of_two(-up) * (scaled ? 1.0f : kLog2E);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      split_pair<PARTS>(to_float(values[s][0]) * power, to_float(values[s][1]) * power, q0[s]);
      split_pair<PARTS>(to_float(values[s][2]) * power, to_float(values[s][3]) * power, q2[s]);
    }
  }
  // From here on this lane deals with the heads 2t and 2t + 1 (columns of the products), with the keys g of every eight.
  const float to_score[2] = {__shfl_sync(0xffffffffu, score_scale, 8 * t), __shfl_sync(0xffffffffu, score_scale, 8 * t + 4)};
  float m[2] = {kQuantLow, kQuantLow}, l[2] = {0.0f, 0.0f};   // the reference, and this lane's share of the sum
  float top[2] = {0.0f, 0.0f}, up[2] = {1.0f, 1.0f};
  float o[HD / 16][4];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  int given_up_at = stages;
  bool begun = false;   // whether a stage has set the reference

  for (int i = 0; i < stages; ++i) {
    const int slot = i % STAGES;
    asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2));
    // Also where every lane's scales of stage i have landed, and every lane is done with stage i - 1. A wait that ran out
    // says so in the status word; what is under way is waited for behind the loop.
    if (!barrier_wait_warp(&landed[slot], (i / STAGES) & 1, a.status)) {
      given_up_at = i;
      break;
    }
    __syncwarp();
    const int next_box = page_of(i + STAGES, box_key), next_scale = page_of(i + STAGES, scale_key);
    issue(i + STAGES - 1, box_page, scale_page);
    box_page = next_box;
    scale_page = next_scale;
    const int key0 = first_of(i);
    if (!holds(key0)) continue;
    unsigned char* at = ring + slot * (2 * Tile::kRowBytes);
    const float* scales = ring_scales + slot * Tile::kScales;

    // ---- scores: eight b, this lane has key b * 8 + g and heads 2t, 2t + 1
    float s[EIGHTS][2];
    {
      float d[2][EIGHTS / 2][4];   // two sums each, so that a product waits for half as many
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int h = 0; h < EIGHTS / 2; ++h) d[x][h][0] = d[x][h][1] = d[x][h][2] = d[x][h][3] = 0.0f;
#pragma unroll
      for (int j = 0; j < Tile::kChunks; ++j) {
        uint32_t words[EIGHTS][4];
#pragma unroll
        for (int b = 0; b < EIGHTS; ++b)
          *reinterpret_cast<uint4*>(words[b]) = *reinterpret_cast<const uint4*>(at + Tile::at(b * 8 + g, key_chunk(j)));
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int n = j * 4 + w;
#pragma unroll
          for (int h = 0; h < EIGHTS / 2; ++h) {
            uint32_t a0, a1, a2, a3;
            code_halves<KIND>(words[2 * h][w], a0, a2);
            code_halves<KIND>(words[2 * h + 1][w], a1, a3);
#pragma unroll
            for (int x = 0; x < PARTS; ++x) quant_mma(d[(PARTS == 2 ? x : w) & 1][h], a0, a1, a2, a3, q0[n][x], q2[n][x]);
          }
        }
      }
#pragma unroll
      for (int b = 0; b < EIGHTS; ++b) {
        const float k_scale = scales[b * 8 + g];
#pragma unroll
        for (int j = 0; j < 2; ++j)   // the factors' product first: the sum times either of them may leave float32 where the score does not
          s[b][j] = (d[0][b / 2][2 * (b & 1) + j] + d[1][b / 2][2 * (b & 1) + j]) * (to_score[j] * k_scale);
      }
    }
    if (scaled) {
#pragma unroll
      for (int b = 0; b < EIGHTS; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[b][j] = capped_score(s[b][j], a.softcap);
          if (BIASED && 2 * t + j < live) s[b][j] += bias_at(a.bias.row(head0 + 2 * t + j), pos - (key0 + b * 8 + g), a.bias.far);
          s[b][j] *= kLog2E;
        }
    }
    if (key0 + KEYS - 1 > pos || key0 < first_key) {   // not every key of the stage is seen
#pragma unroll
      for (int b = 0; b < EIGHTS; ++b)
        if (!key_seen(key0 + b * 8 + g, pos, first_key, a.keep)) s[b][0] = s[b][1] = -INFINITY;
    }
    float weight[EIGHTS][2];
    float sum[2], widest[2];
    for (bool anew = !begun;; anew = true) {   // once more where the weights outgrew their room: with a new reference
      float carry[2] = {1.0f, 1.0f};
      if (anew) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float most = m[j];
#pragma unroll
          for (int b = 0; b < EIGHTS; ++b) most = fmaxf(most, s[b][j]);
#pragma unroll
          for (int offset = 4; offset < 32; offset <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, offset));
          carry[j] = quant_exp2<T>(m[j] - most);   // what was gathered so far, on the new reference
          m[j] = most;
        }
      }
      sum[0] = sum[1] = widest[0] = widest[1] = 0.0f;
#pragma unroll
      for (int b = 0; b < EIGHTS; ++b) {
        const float v_scale = scales[KEYS + b * 8 + g];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float p = quant_exp2<T>(s[b][j] - m[j]);
          sum[j] += p;
          weight[b][j] = p * v_scale;
          widest[j] = fmaxf(widest[j], fabsf(weight[b][j]));   // a pool of a caller's own may have scales of either sign
        }
      }
      if (!anew) {
        const bool outgrown = fmaxf(sum[0], sum[1]) > 65536.0f || fmaxf(widest[0] * up[0], widest[1] * up[1]) >= 32768.0f;
        if (!__any_sync(0xffffffffu, outgrown)) break;
        continue;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float most = widest[j];
#pragma unroll
        for (int offset = 4; offset < 32; offset <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, offset));
        top[j] = fmaxf(top[j] * carry[j], most);
        const float before = up[j];
        // 2^125 at most, whose reciprocal __fdividef still gives (beyond 2^126 it gives 0)
        up[j] = power_of_two(min(kQuantTop - (static_cast<int>(__float_as_uint(top[j]) >> 23) - 127), 125));
        // a quotient beyond float32 means that what was gathered is nothing on the new reference: carry is 0 then
        const float factor = carry[j] * fminf(up[j] / before, 0x1p127f);
        l[j] *= carry[j];
        if (begun) {
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) { o[n][j] *= factor; o[n][2 + j] *= factor; }
        }
      }
      begun = true;
      break;
    }
    l[0] += sum[0];
    l[1] += sum[1];
    uint32_t p[EIGHTS][PARTS];   // keys b * 8 + 2t, 2t + 1 of head g
#pragma unroll
    for (int b = 0; b < EIGHTS; ++b) {
      split_pair<PARTS>(weight[b][0] * up[0], weight[b][1] * up[1], p[b]);
#pragma unroll
      for (int x = 0; x < PARTS; ++x) p[b][x] = turn_tile(p[b][x]);
    }
    // ---- o^T += V^T p^T, sixteen keys at a time
    at += Tile::kRowBytes;
    if (key0 + KEYS - 1 > pos || key0 < first_key) {
      // A key that is not seen has weight 0, but 0 x NaN is NaN: whatever its page's earlier owner left becomes zeros.
      const int r = lane % KEYS, key = key0 + r;
      if (!key_seen(key, pos, first_key, a.keep))
        for (int c = lane / KEYS; c < HD / 16; c += 32 / KEYS) *reinterpret_cast<uint4*>(at + Tile::at(r, c)) = make_uint4(0u, 0u, 0u, 0u);
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");   // ahead of the copy that fills the slot next
      __syncwarp();
    }
#pragma unroll
    for (int h = 0; h < KEYS / 16; ++h) {
#pragma unroll
      for (int j = 0; j < Tile::kValuePieces; ++j) {
        constexpr int WORDS = Tile::kValueBytes / 4;
        uint32_t v[4][WORDS];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int r = h * 16 + 2 * t + (n & 1) + (n >> 1) * 8;
          const unsigned char* src = at + (HD == 64 ? Tile::at(r, g >> 1) + (g & 1) * 8 : Tile::at(r, j * 8 + g));
          if (WORDS == 4) *reinterpret_cast<uint4*>(v[n]) = *reinterpret_cast<const uint4*>(src);
          else *reinterpret_cast<uint2*>(v[n]) = *reinterpret_cast<const uint2*>(src);
        }
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {   // values 2 half and 2 half + 1 of the word: bytes of keys 2t, 2t + 1 side by side
            const uint32_t pick = half ? 0x7362 : 0x5140;
            uint32_t a0, a1, a2, a3;
            code_halves<KIND>(__byte_perm(v[0][w], v[1][w], pick), a0, a1);
            code_halves<KIND>(__byte_perm(v[2][w], v[3][w], pick), a2, a3);
#pragma unroll
            for (int x = 0; x < PARTS; ++x) quant_mma(o[j * 2 * WORDS + 2 * w + half], a0, a1, a2, a3, p[2 * h][x], p[2 * h + 1][x]);
          }
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::);
  for (int i = given_up_at; i < stages && i < given_up_at + STAGES - 1; ++i)   // a warp that gives up waits for its copies under way
    barrier_wait_warp(&landed[i % STAGES], (i / STAGES) & 1, a.status);
#pragma unroll
  for (int offset = 4; offset < 32; offset <<= 1) {
    l[0] += __shfl_xor_sync(0xffffffffu, l[0], offset);
    l[1] += __shfl_xor_sync(0xffffffffu, l[1], offset);
  }
  if (release_late) chain_release();

  // ---- the four warps in warp order: this block's partial result (the area lies over the ring, which is used up)
  __syncthreads();
  float* merge = reinterpret_cast<float*>(quant_shared);   // [warps][8 heads][HD + 2]
  {
    const float d0 = __fdividef(1.0f, up[0]), d1 = __fdividef(1.0f, up[1]);   // powers of two
#pragma unroll
    for (int n = 0; n < HD / 16; ++n) {
      constexpr int BLOCKS = Tile::kValueBytes / 2;   // of 16 values, from one piece
      const int d = (n / BLOCKS) * 128 + g * Tile::kValueBytes + (n % BLOCKS) * 2;
      float* to = merge + (warp * 8 + 2 * t) * (HD + 2) + d;
      *reinterpret_cast<float2*>(to) = make_float2(o[n][0] * d0, o[n][2] * d0);
      *reinterpret_cast<float2*>(to + HD + 2) = make_float2(o[n][1] * d1, o[n][3] * d1);
    }
  }
  if (g == 0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      merge[(warp * 8 + 2 * t + j) * (HD + 2) + HD] = m[j];
      merge[(warp * 8 + 2 * t + j) * (HD + 2) + HD + 1] = l[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < live * HD; i += kDecodeThreads) {
    const int h = i / HD, d = i - h * HD;
    float m_all = kQuantLow;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m_all = fmaxf(m_all, merge[(w * 8 + h) * (HD + 2) + HD]);
    float sum = 0.0f, l_all = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float* theirs = merge + (w * 8 + h) * (HD + 2);
      const float weight = quant_exp2<T>(theirs[HD] - m_all);   // a warp without keys has l = 0 and zeros
      sum += weight * theirs[d];
      l_all += weight * theirs[HD + 1];
    }
    float* dst = a.fused ? results + h * (HD + 2) : a.partial + ((static_cast<size_t>(row) * a.heads + head0 + h) * slots + rank) * (HD + 2);
    dst[d] = sum;
    if (d == 0) { dst[HD] = a.fused ? m_all : m_all * 0.6931471805599453f; dst[HD + 1] = l_all; }   // the merge kernel works in natural units
  }
  if (a.fused) finish();
}

// Whether the tensor-core kernel takes these rows: pieces of 16 bytes (queries: 8 or 16) that lie on such boundaries, and
// pages of a power of two of 8 positions or more.
static bool quantized_mma_takes(const QuantizedDecode& a) {
  return a.page_shift >= 3 && (a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) && reinterpret_cast<uintptr_t>(a.codes) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(a.q) % 16 == 0;
}

// How many blocks a (token, key/value head) pair gets of the tensor-core kernel, `tiles` being the most that one has and
// `resident` how many blocks the GPU holds. Where that leaves blocks eight tiles or more, two rounds of blocks: the contexts of
// a batch differ, and blocks of the longest would be alone for half the time. With 8 key/value heads and contexts spread
// evenly up to 36,000 positions (heads of 128, four to a key/value head; us in one round and in two): 4 requests 43 and 40,
// 8 requests 73 and 60, 16 requests 135 and 102; contexts of one length pay for it: 8 of 32,000 86 and 89, 16 of 8,000 47
// and 52. From four tiles a block on, 8 of 8,000 would go from 28 to 31, and few ragged requests (3 to 16 with 1 to 8 key/value
// heads) gain or lose 1 us or less.
// Else one round, and two tiles a block from 32 tiles on (1 of 8,000: 11.2, with one tile a block 12.6).
static int quantized_slots(int pairs, int tiles, int resident) {
  const int twice = pairs <= resident ? 2 * resident / pairs : (2 * resident + pairs / 2) / pairs;
  if (pairs > 1 && twice > 1 && tiles >= 8 * twice) return twice;
  int slots = resident / pairs;
  const int most = tiles <= 16 ? tiles : (tiles / 2 > 16 ? tiles / 2 : 16);
  if (slots > most) slots = most;
  return slots > 1 ? slots : 1;
}

template <typename T, int KIND, int HD>
static cudaError_t launch_quantized_mma(const QuantizedDecode& args, dim3 grid, cudaStream_t stream) {
  auto kernel = args.bias.table != nullptr ? quantized_decode_mma_kernel<T, KIND, HD, true> : quantized_decode_mma_kernel<T, KIND, HD, false>;
  if (QuantTile<HD>::kShared > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, QuantTile<HD>::kShared);
    if (e != cudaSuccess) return e;
  }
  CUtensorMap map;
  const int keys = QuantTile<HD>::kKeys;
  if (!encode_codes_map(&map, args.codes, static_cast<long long>(args.num_pages) * 2 * args.kv_heads * args.page_tokens, HD,
                        args.page_tokens < keys ? args.page_tokens : keys))
    return cudaErrorInvalidValue;
  if (args.fused && grid.x > 1) return launch_chained_clusters(kernel, grid, dim3(kDecodeThreads), QuantTile<HD>::kShared, grid.x, stream, map, args);
  return launch_chained(kernel, grid, dim3(kDecodeThreads), QuantTile<HD>::kShared, stream, map, args);
}

// Launches the kernel that takes the shape; `slots` says into how many partial results a pair was cut, 0 that the output
// is made. `fusable`: the caller wants the output, not the partial results. Without room for them: cudaErrorNotReady if they
// are needed, and nothing is launched.
constexpr int kQuantCluster = 8;   // blocks of a cluster, at most
template <typename T>
static cudaError_t launch_quantized_decode(QuantizedDecode args, int kind, int rows, bool fusable, int* slots, cudaStream_t stream) {
  const int parts = (args.heads / args.kv_heads + kQuantHeads - 1) / kQuantHeads, pairs = rows * args.kv_heads * parts;
  int tiles = args.max_splits;   // the most that a pair has
  if (args.window > 0) tiles = min(tiles, (args.window + kSplitKeys - 1) / kSplitKeys + 1 + (args.keep + kSplitKeys - 1) / kSplitKeys);
  if (args.chunk > 0) tiles = min(tiles, (args.chunk + kSplitKeys - 1) / kSplitKeys + 1 + (args.keep + kSplitKeys - 1) / kSplitKeys);
  if (quantized_mma_takes(args)) {
    const int resident = 148 * (args.head_dim == 256 ? QuantBlocks<T, 256>::value : QuantBlocks<T, 128>::value);
    int count = quantized_slots(pairs, tiles, resident);
    // Few tiles over a few more blocks than a cluster has: the launch and the trip through memory that the merge kernel
    // costs are worth more than the blocks (4 requests of 2,048 positions 8.2 us, else 10.4; 4 of 5,000 14.0 and 14.9; but 1
    // of 4,096 9.6 and 8.5). Not with longer contexts: 1 of 8,000 would go from 11.2 to 13.9.
    if (fusable && count > kQuantCluster && tiles <= 6 * kQuantCluster && kQuantCluster * pairs <= resident) count = kQuantCluster;
    // Clusters only where all blocks are resident at once: in further rounds a cluster waits for as many places side by side
    // (37 requests of 7,000 positions in three blocks a pair: 115 us as clusters, 92 without).
    args.fused = fusable && (count == 1 || (count <= kQuantCluster && static_cast<long long>(count) * pairs <= resident));
    if (!args.fused && args.partial == nullptr) return cudaErrorNotReady;   // the caller is to bring room for the partial results
    *slots = args.fused ? 0 : count;
    const dim3 grid(count, args.kv_heads * parts, rows);
#define BY_SIZE(KIND) (args.head_dim == 64    ? launch_quantized_mma<T, KIND, 64>(args, grid, stream)  \
                       : args.head_dim == 128 ? launch_quantized_mma<T, KIND, 128>(args, grid, stream) \
                                              : launch_quantized_mma<T, KIND, 256>(args, grid, stream))
    return kind == kCodesInt8 ? BY_SIZE(kCodesInt8) : BY_SIZE(kCodesE4M3);
#undef BY_SIZE
  }
  if (args.partial == nullptr) return cudaErrorNotReady;
  *slots = max(1, min(kDecodeBlocksAtOnce / static_cast<unsigned>(pairs), static_cast<unsigned>(args.max_splits)));
  const dim3 grid(*slots, args.kv_heads * parts, rows);
  auto launch = [&](auto kernel) {
    kernel<<<grid, kDecodeThreads, 0, stream>>>(args);
    return cudaGetLastError();
  };
#define BY_KIND(VALUES) (kind == kCodesInt8 ? launch(quantized_decode_kernel<T, kCodesInt8, VALUES>) \
                                            : launch(quantized_decode_kernel<T, kCodesE4M3, VALUES>))
  if (args.head_dim <= 64) return BY_KIND(2);
  if (args.head_dim <= 128) return BY_KIND(4);
  return BY_KIND(8);
#undef BY_KIND
}

}  // namespace mxb
