// Attention of single decoded tokens over a cache held in 8 bits (the rows of
// quantized.cuh): scores s_j = (q . code_j) scale_j, softmax, and the sum of
// (p_j scale_j) code_j, in float32, without ever making the rows themselves.
//
// Work is cut as the kernels over a cache in the compute type cut it: a pair of
// (token, key/value head) gets `slots` blocks, block s takes the tiles of
// kSplitKeys keys first + s, first + s + slots, ... of the token's keys and leaves
// one unnormalised partial result (accumulator, maximum, sum), which the merge
// kernel puts together in slot order.
#pragma once

#include <cuda_fp16.h>

#include "quantized.cuh"

namespace mxb {

struct QuantizedDecode {
  const void* q;                 // [tokens, heads, head_dim]
  const uint8_t* codes;
  const float* scales;
  float* partial;                // [rows, heads, slots, head_dim + 2]
  const int* block_tables;
  int max_pages;
  const int *row_token, *row_request, *positions;
  int heads, kv_heads, head_dim, page_tokens, num_pages, window, chunk, keep;
  float scale, softcap;
  ScoreBias bias;
  int page_shift;                // log2 of page_tokens, -1 where that is no power of two
  int settled;                   // the positions ahead of each token's own were written by launches before the last one
  int* status;
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
        k[i] = d < n ? code_value<KIND>(a.codes[k_row * n + d]) : 0.0f;
        v[i] = d < n ? code_value<KIND>(a.codes[v_row * n + d]) : 0.0f;
      }
#pragma unroll
      for (int h = 0; h < G; ++h) {
        if (h >= live) continue;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) s = fmaf(q[h][i], k[i], s);
        s = capped_score(warp_sum(s) * k_scale * a.scale, a.softcap);
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
// 2^-39 of it), and the weights p_j scale_j so that the largest so far does.
// With `top` the largest such weight on the running maximum's terms, ref = 2^floor(log2 top),
// the accumulator holds sum_j (2^14 / ref) p_j scale_j code_j.
//
// A warp works alone until the end: it takes its 32 keys of a 128-key tile (a
// stage; for heads of 256, 16 of them), copies their rows into a ring of its own
// by cp.async, each lane exactly the pieces that it will read itself, and so needs
// neither a barrier nor a bank's favour: a lane's 16 bytes lie beside its
// neighbours'. What a lane reads is chosen so that bytes need no transposing:
//   K: lane (g, t) = (lane / 4, lane % 4) of the key g of eight copies the 16-byte
//      pieces t, t + 4, ... of that row. Word w of a piece gives both registers
//      of the B operand of one 16-value step; q's registers follow the same
//      order of values.
//   V: lane (g, t) copies 16 bytes at g of the rows of the keys 2t, 2t + 1, 2t + 8,
//      2t + 9, from which byte pairs of neighbouring keys make the A operand
//      (o^T = V^T p^T: 16 values of a row by 8 query heads, no row of the tile
//      wasted). The scores lie where p^T's B operand wants them.
//
// float32 queries are two halves each, 22 bits and the sign of what is left (the
// second as rows 8..15 of the same product); so are the weights, in a product more.
template <int HD> struct QuantTile {
  static constexpr int kKeys = HD == 256 ? 16 : 32;            // of a stage
  static constexpr int kBlocks8 = kKeys / 8;                   // eights of keys
  static constexpr int kKeyPieces = HD / 64;                   // 16-byte pieces of a key row a lane takes
  static constexpr int kValueBytes = HD >= 128 ? 16 : HD / 8;  // of a value row a lane takes at once
  static constexpr int kValuePieces = HD / 8 / kValueBytes;
  static constexpr int kRowBytes = kKeys * HD;                 // a stage's keys; its values as many
  static constexpr int kStageBytes = 2 * kRowBytes + 2 * kKeys * 4;   // keys, values, scales
  static constexpr int kStages = HD == 128 ? 2 : 3;
  static constexpr int kRing = (kDecodeThreads / 32) * kStages * kStageBytes;
  static constexpr int kMerge = (kDecodeThreads / 32) * 8 * (HD + 2) * 4;
  static constexpr int kShared = kRing > kMerge ? kRing : kMerge;
};

template <int BYTES> __device__ __forceinline__ void quant_copy(void* dst, const void* src, bool there) {
  const uint32_t address = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  const int size = there ? BYTES : 0;   // else zeros
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(address), "l"(src), "r"(size));
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(address), "l"(src), "n"(BYTES), "r"(size));
}

// The four codes of a word as two pairs of halves. Whole numbers: with its sign
// bit turned a code is an unsigned u = code + 128, and the half with the bits
// 0x6400 + u is 1024 + u.
template <int KIND> __device__ __forceinline__ void code_halves(uint32_t word, uint32_t& lower, uint32_t& upper) {
  if (KIND == kCodesE4M3) {
    asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\ncvt.rn.f16x2.e4m3x2 %0, lo;\ncvt.rn.f16x2.e4m3x2 %1, hi;\n}\n"
        : "=r"(lower), "=r"(upper) : "r"(word));
  } else {
    const uint32_t turned = word ^ 0x80808080u, off = 0xe480e480u;   // -1152
    const __half2 less = *reinterpret_cast<const __half2*>(&off);
    const uint32_t lo = __byte_perm(turned, 0x64646464u, 0x4140), hi = __byte_perm(turned, 0x64646464u, 0x4342);
    const __half2 a = __hadd2(*reinterpret_cast<const __half2*>(&lo), less), b = __hadd2(*reinterpret_cast<const __half2*>(&hi), less);
    lower = *reinterpret_cast<const uint32_t*>(&a);
    upper = *reinterpret_cast<const uint32_t*>(&b);
  }
}

__device__ __forceinline__ void quant_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// Blocks resident on an SM: what the ring and the registers leave room for.
template <typename T, int HD> struct QuantBlocks {
  static constexpr int value = HD == 256 ? (std::is_same<T, float>::value ? 1 : 2) : 3;
};

template <typename T, int KIND, int HD, bool BIASED>
__global__ void __launch_bounds__(kDecodeThreads, QuantBlocks<T, HD>::value)
quantized_decode_mma_kernel(const QuantizedDecode a) {
  using Tile = QuantTile<HD>;
  constexpr int PARTS = std::is_same<T, float>::value ? 2 : 1;
  constexpr int WARPS = kDecodeThreads / 32, STAGES = Tile::kStages, STEPS = HD / 16, KEYS = Tile::kKeys, EIGHTS = Tile::kBlocks8;
  constexpr int HALVES = 32 / KEYS;   // stages of a warp's 32 keys of a tile
  constexpr float kLog2E = 1.4426950408889634f;
  extern __shared__ __align__(16) unsigned char quant_shared[];
  const bool release_late = gridDim.x * gridDim.y * gridDim.z > QuantBlocks<T, HD>::value * 148u;   // as in the kernels over bfloat16 rows
  if (!release_late) chain_release();
  const int rank = blockIdx.x, slots = gridDim.x, kv = blockIdx.y % a.kv_heads, part = blockIdx.y / a.kv_heads, row = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  if (!a.settled) chain_wait();
  const int token = a.row_token[row];
  if (token < 0) return;   // a padding row
  const int pos = a.positions[token], group = a.heads / a.kv_heads;
  const int live = min(group - part * 8, 8), head0 = kv * group + part * 8;   // this block's query heads
  const int first_key = first_visible_key(pos, a.window, a.chunk);
  const KeyWalk walk = key_walk(first_key, pos, a.keep, kSplitKeys);
  if (rank >= walk.count) return;   // more slots than tiles: the merge skips this one
  const int* table = a.block_tables + static_cast<size_t>(a.row_request[row]) * a.max_pages;
  unsigned char* ring = quant_shared + warp * (STAGES * Tile::kStageBytes);

  // Stage i of the warp: part i % HALVES of its keys of the block's tile i / HALVES.
  const int stages = HALVES * ((walk.count - rank + slots - 1) / slots);
  auto first_of = [&](int i) { return walk.tile(rank + i / HALVES * slots) * kSplitKeys + warp * 32 + i % HALVES * KEYS; };
  auto holds = [&](int key0) { return key0 <= pos && (key0 + KEYS > first_key || key0 < a.keep); };
  // Pages are a power of two of 8 positions or more, so eight keys lie in one of them. Lanes b, b + 4, ... ask for the page
  // of eight b of a stage, one stage ahead of the copies, and look at it only then.
  const int shift = a.page_shift, in_page = a.page_tokens - 1;
  auto page_of = [&](int i) {
    const int slot = (first_of(i) + lane % EIGHTS * 8) >> shift;
    return i < stages && slot < a.max_pages ? table[slot] : -1;
  };
  const int value_rows = a.kv_heads * a.page_tokens;   // from a key's row to its value's
  const uint8_t* k_lane = a.codes + g * HD + t * 16;
  const uint8_t* v_lane = a.codes + (static_cast<size_t>(value_rows) + 2 * t) * HD + g * Tile::kValueBytes;
  auto copies = [&](int i, int key0, int page, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;   // every key of the stage is seen
    unsigned char* at = ring + (i % STAGES) * Tile::kStageBytes;
    const int key8 = key0 + lane % EIGHTS * 8;
    bool there = page >= 0 && page < a.num_pages;
    if (!there && key8 <= pos && (key8 + 8 > first_key || key8 < a.keep)) atomicOr(a.status, kStatusBadPage);
    const int base = there ? (page * 2 * a.kv_heads + kv) * a.page_tokens + (key8 & in_page) : -1;   // the pool row of the eight's first key
    auto seen = [&](int key) { return WHOLE || key_seen(key, pos, first_key, a.keep); };
#pragma unroll
    for (int b = 0; b < EIGHTS; ++b) {
      const int from = __shfl_sync(0xffffffffu, base, b);
      const size_t offset = static_cast<size_t>(max(from, 0)) * HD;
      const bool k_there = from >= 0 && seen(key0 + b * 8 + g);
#pragma unroll
      for (int j = 0; j < Tile::kKeyPieces; ++j)
        quant_copy<16>(at + ((b * Tile::kKeyPieces + j) * 32 + lane) * 16, k_lane + offset + j * 64, k_there);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const bool v_there = from >= 0 && seen(key0 + b * 8 + 2 * t + n);
#pragma unroll
        for (int j = 0; j < Tile::kValuePieces; ++j)
          quant_copy<Tile::kValueBytes>(at + Tile::kRowBytes + (((b * 2 + n) * Tile::kValuePieces + j) * 32 + lane) * Tile::kValueBytes,
                                        v_lane + offset + n * HD + j * 128, v_there);
      }
    }
    // a lane a key for the scales (heads of 256: lanes 16 to 31 the values')
    const int key = lane % KEYS, from = __shfl_sync(0xffffffffu, base, key >> 3);
    there = from >= 0 && seen(key0 + key);
    const float* scale = a.scales + max(from, 0) + (key & 7);
    at += 2 * Tile::kRowBytes;
    if (KEYS == 32) {
      quant_copy<4>(at + lane * 4, scale, there);
      quant_copy<4>(at + (32 + lane) * 4, scale + value_rows, there);
    } else {
      quant_copy<4>(at + lane * 4, scale + (lane < KEYS ? 0 : value_rows), there);
    }
  };
  auto issue = [&](int i, int page) {
    const int key0 = first_of(i);
    if (i < stages && holds(key0)) {
      if (key0 >= first_key && key0 + KEYS - 1 <= pos) copies(i, key0, page, std::true_type());
      else copies(i, key0, page, std::false_type());
    }
    asm volatile("cp.async.commit_group;\n" ::);
  };
  // The token's own row, of the walk's last tile, is written by the kernel ahead of this one; with `settled` all others
  // are older, and their copies start ahead of the wait.
  bool waited = !a.settled;
  int page = page_of(0);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (!waited && i < stages && first_of(i) + KEYS > pos) {
      chain_wait();
      waited = true;
    }
    const int next_page = page_of(i + 1);
    issue(i, page);
    page = next_page;
  }
  if (!waited) chain_wait();

  // ---- the query heads as rows 0..7 (float32: their second halves as rows 8..15)
  const bool scaled = BIASED || a.softcap > 0.0f;   // scores in natural units first; else in powers of two at once
  uint32_t q0[STEPS][PARTS], q2[STEPS][PARTS];
  float score_scale;
  {
    const T* q = behind_wait(static_cast<const T*>(a.q)) + (static_cast<size_t>(token) * a.heads + head0 + (g < live ? g : 0)) * HD;
    alignas(16) T values[STEPS][4];
    uint32_t largest = 0;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const T* at = q + (s >> 2) * 64 + t * 16 + (s & 3) * 4;
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
  float m_run = -INFINITY, l_run = 0.0f;   // of head g, over this warp's keys so far; the sum over this lane's alone
  float top = 0.0f;
  int ref = -100;                          // exponent of the reference, 2^floor(log2 top) but not below 2^-100
  float o[HD / 16][4];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

  for (int i = 0; i < stages; ++i) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2));
    __syncwarp();   // every lane's copies of stage i have landed, and every lane is done with stage i - 1
    const int next_page = page_of(i + STAGES);
    issue(i + STAGES - 1, page);
    page = next_page;
    const int key0 = first_of(i);
    if (!holds(key0)) continue;
    const unsigned char* at = ring + (i % STAGES) * Tile::kStageBytes;
    const float* scales = reinterpret_cast<const float*>(at + 2 * Tile::kRowBytes);

    // ---- scores: this lane has those of head g and keys b * 8 + 2t, 2t + 1
    float s[EIGHTS][2];
    float d[EIGHTS][4];
#pragma unroll
    for (int b = 0; b < EIGHTS; ++b) d[b][0] = d[b][1] = d[b][2] = d[b][3] = 0.0f;
#pragma unroll
    for (int j = 0; j < Tile::kKeyPieces; ++j) {
      uint32_t words[EIGHTS][4];
#pragma unroll
      for (int b = 0; b < EIGHTS; ++b)
        *reinterpret_cast<uint4*>(words[b]) = *reinterpret_cast<const uint4*>(at + ((b * Tile::kKeyPieces + j) * 32 + lane) * 16);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int n = j * 4 + w;
#pragma unroll
        for (int b = 0; b < EIGHTS; ++b) {   // the eights' sums do not wait for one another
          uint32_t b0, b1;
          code_halves<KIND>(words[b][w], b0, b1);
          quant_mma(d[b], q0[n][0], PARTS == 2 ? q0[n][PARTS - 1] : 0u, q2[n][0], PARTS == 2 ? q2[n][PARTS - 1] : 0u, b0, b1);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < EIGHTS; ++b) {
      const float2 k_scale = *reinterpret_cast<const float2*>(scales + b * 8 + 2 * t);
      s[b][0] = (PARTS == 2 ? d[b][0] + d[b][2] : d[b][0]) * score_scale * k_scale.x;
      s[b][1] = (PARTS == 2 ? d[b][1] + d[b][3] : d[b][1]) * score_scale * k_scale.y;
    }
    if (scaled) {
#pragma unroll
      for (int b = 0; b < EIGHTS; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[b][j] = capped_score(s[b][j], a.softcap);
          if (BIASED && g < live) s[b][j] += bias_at(a.bias.row(head0 + g), pos - (key0 + b * 8 + 2 * t + j), a.bias.far);
          s[b][j] *= kLog2E;
        }
    }
    if (key0 + KEYS - 1 > pos || key0 < first_key) {   // not every key of the stage is seen
#pragma unroll
      for (int b = 0; b < EIGHTS; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (!key_seen(key0 + b * 8 + 2 * t + j, pos, first_key, a.keep)) s[b][j] = -INFINITY;
    }
    float m_new = m_run;
#pragma unroll
    for (int b = 0; b < EIGHTS; ++b) m_new = fmaxf(m_new, fmaxf(s[b][0], s[b][1]));
    m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 1));
    m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 2));
    const float zero = m_new == -INFINITY ? 0.0f : m_new;
    const float carry = quant_exp2<T>(m_run - zero);   // what earlier stages gathered, on the new maximum (0 if nothing yet)
    float l_new = 0.0f, widest = 0.0f;
#pragma unroll
    for (int b = 0; b < EIGHTS; ++b) {
      const float p0 = quant_exp2<T>(s[b][0] - zero), p1 = quant_exp2<T>(s[b][1] - zero);
      l_new += p0 + p1;
      const float2 v_scale = *reinterpret_cast<const float2*>(scales + KEYS + b * 8 + 2 * t);
      s[b][0] = p0 * v_scale.x;
      s[b][1] = p1 * v_scale.y;
      widest = fmaxf(widest, fmaxf(s[b][0], s[b][1]));
    }
    l_run = l_run * carry + l_new;
    widest = fmaxf(widest, __shfl_xor_sync(0xffffffffu, widest, 1));
    widest = fmaxf(widest, __shfl_xor_sync(0xffffffffu, widest, 2));
    top = fmaxf(top * carry, widest);
    const int ref_new = max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100);
    const bool moved = m_new != m_run || ref_new != ref;
    if (__any_sync(0xffffffffu, moved)) {
      const float factor = moved ? carry * power_of_two(max(min(ref - ref_new, 127), -126)) : 1.0f;
      const float c0 = __shfl_sync(0xffffffffu, factor, 8 * t), c1 = __shfl_sync(0xffffffffu, factor, 8 * t + 4);   // heads 2t, 2t + 1
#pragma unroll
      for (int n = 0; n < HD / 16; ++n) { o[n][0] *= c0; o[n][1] *= c1; o[n][2] *= c0; o[n][3] *= c1; }
    }
    m_run = m_new;
    ref = ref_new;
    const float up = power_of_two(14 - ref);
    uint32_t p[EIGHTS][PARTS];   // the weights of key pairs b * 8 + 2t, 2t + 1, times the values' scales
#pragma unroll
    for (int b = 0; b < EIGHTS; ++b) split_pair<PARTS>(s[b][0] * up, s[b][1] * up, p[b]);
    // ---- o^T += V^T p^T, sixteen keys at a time
    at += Tile::kRowBytes;
#pragma unroll
    for (int h = 0; h < KEYS / 16; ++h) {
#pragma unroll
      for (int j = 0; j < Tile::kValuePieces; ++j) {
        constexpr int WORDS = Tile::kValueBytes / 4;
        uint32_t v[4][WORDS];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const unsigned char* src = at + (((h * 4 + n) * Tile::kValuePieces + j) * 32 + lane) * Tile::kValueBytes;
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
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
  if (release_late) chain_release();

  // ---- the four warps in warp order: this block's partial result (the area lies over the ring, which is used up)
  __syncthreads();
  float* merge = reinterpret_cast<float*>(quant_shared);   // [warps][8 heads][HD + 2]
  {
    const float down = power_of_two(ref - 14), d0 = __shfl_sync(0xffffffffu, down, 8 * t), d1 = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
    for (int n = 0; n < HD / 16; ++n) {
      constexpr int BLOCKS = Tile::kValueBytes / 2;   // of 16 values, from one piece
      const int d = (n / BLOCKS) * 128 + g * Tile::kValueBytes + (n % BLOCKS) * 2;
      float* to = merge + (warp * 8 + 2 * t) * (HD + 2) + d;
      *reinterpret_cast<float2*>(to) = make_float2(o[n][0] * d0, o[n][2] * d0);
      *reinterpret_cast<float2*>(to + HD + 2) = make_float2(o[n][1] * d1, o[n][3] * d1);
    }
  }
  if (t == 0) {
    merge[(warp * 8 + g) * (HD + 2) + HD] = m_run;
    merge[(warp * 8 + g) * (HD + 2) + HD + 1] = l_run;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < live * HD; i += kDecodeThreads) {
    const int h = i / HD, d = i - h * HD;
    float m_all = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m_all = fmaxf(m_all, merge[(w * 8 + h) * (HD + 2) + HD]);
    float sum = 0.0f, l_all = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float* theirs = merge + (w * 8 + h) * (HD + 2);
      const float weight = quant_exp2<T>(theirs[HD] - m_all);   // a warp without keys has m = -inf: weight 0
      sum += weight * theirs[d];
      l_all += weight * theirs[HD + 1];
    }
    float* dst = a.partial + ((static_cast<size_t>(row) * a.heads + head0 + h) * slots + rank) * (HD + 2);
    dst[d] = sum;
    if (d == 0) { dst[HD] = m_all * 0.6931471805599453f; dst[HD + 1] = l_all; }   // the merge kernel works in natural units
  }
}

// Whether the tensor-core kernel takes these rows: pieces of 16 bytes (queries: 8 or 16) that lie on such boundaries, and
// pages of a power of two of 8 positions or more.
static bool quantized_mma_takes(const QuantizedDecode& a) {
  return a.page_shift >= 3 && (a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) && reinterpret_cast<uintptr_t>(a.codes) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(a.q) % 16 == 0;
}

// How many blocks a (token, key/value head) pair gets: as many as fill the GPU
// with blocks resident at once, no more than it has tiles.
static int quantized_slots(int pairs, int max_splits, int resident) {
  int wanted = pairs > 0 ? resident / pairs : 1;
  if (wanted < 1) wanted = 1;
  return wanted < max_splits ? wanted : max_splits;
}

template <typename T, int KIND, int HD>
static cudaError_t launch_quantized_mma(const QuantizedDecode& args, dim3 grid, cudaStream_t stream) {
  auto kernel = args.bias.table != nullptr ? quantized_decode_mma_kernel<T, KIND, HD, true> : quantized_decode_mma_kernel<T, KIND, HD, false>;
  if (QuantTile<HD>::kShared > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, QuantTile<HD>::kShared);
    if (e != cudaSuccess) return e;
  }
  return launch_chained(kernel, grid, dim3(kDecodeThreads), QuantTile<HD>::kShared, stream, args);
}

// Launches the kernel that takes the shape; `slots` says into how many partial results a pair was cut.
template <typename T>
static cudaError_t launch_quantized_decode(const QuantizedDecode& args, int kind, int rows, int max_splits, int* slots, cudaStream_t stream) {
  const int parts = (args.heads / args.kv_heads + kQuantHeads - 1) / kQuantHeads, pairs = rows * args.kv_heads * parts;
  if (quantized_mma_takes(args)) {
    *slots = quantized_slots(pairs, max_splits, 148 * (args.head_dim == 256 ? QuantBlocks<T, 256>::value : QuantBlocks<T, 128>::value));
    const dim3 grid(*slots, args.kv_heads * parts, rows);
#define BY_SIZE(KIND) (args.head_dim == 64    ? launch_quantized_mma<T, KIND, 64>(args, grid, stream)  \
                       : args.head_dim == 128 ? launch_quantized_mma<T, KIND, 128>(args, grid, stream) \
                                              : launch_quantized_mma<T, KIND, 256>(args, grid, stream))
    return kind == kCodesInt8 ? BY_SIZE(kCodesInt8) : BY_SIZE(kCodesE4M3);
#undef BY_SIZE
  }
  *slots = quantized_slots(pairs, max_splits, kDecodeBlocksAtOnce);
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
