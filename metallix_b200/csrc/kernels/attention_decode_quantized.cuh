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
// either kind are exact in bfloat16, so the products q . code and p . code are
// mma.sync m16n8k16 with float32 sums, the scales joining behind and ahead of
// them. Bound by the codes' bytes where contexts are long, and by its start-up
// where they are short; what it is built for is to keep many bytes on their way
// with few instructions per byte.
//
// A warp works alone until the end: it takes 16 keys at a time (a stage) of its
// 32 of every 128-key tile, copies their rows into a ring of its own by
// cp.async, each lane exactly the pieces that it will read itself, and so needs
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
// float32 queries are three bfloat16 parts each, which hold their 24 bits (the
// first two as rows 0..7 and 8..15 of one product); so are the weights.
template <int HD> struct QuantTile {
  static constexpr int kKeys = 16;                             // of a stage
  static constexpr int kKeyPieces = HD / 64;                   // 16-byte pieces of a key row a lane takes
  static constexpr int kValueBytes = HD >= 128 ? 16 : HD / 8;  // of a value row a lane takes at once
  static constexpr int kValuePieces = HD / 8 / kValueBytes;
  static constexpr int kRowBytes = 2 * kKeyPieces * 16 * 32;   // a stage's keys, over the warp: two rows a lane
  static constexpr int kStageBytes = kRowBytes + 4 * kValuePieces * kValueBytes * 32 + 2 * kKeys * 4;   // and values, four a lane, and scales
  static constexpr int kStages = HD == 64 ? 4 : 3;
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

// Two codes, the bytes `pick` names of a and b, as a pair of bfloat16 numbers.
// e4m3: sign and the seven bits of the magnitude move to where bfloat16 has
// them, which leaves the number 2^-120 times too small (small e4m3 numbers
// become small bfloat16 ones). Whole numbers: 128 + the low seven bits, less
// 128, or 256 for a negative one.
template <int KIND> __device__ __forceinline__ uint32_t code_pair(uint32_t a, uint32_t b, uint32_t pick) {
  const uint32_t x = __byte_perm(a, b, pick);   // each code in both bytes of its half
  __nv_bfloat162 out;
  if (KIND == kCodesE4M3) {
    const uint32_t bits = (x & 0x80008000u) | ((x >> 4) & 0x07f007f0u);
    const uint32_t up = 0x7b807b80u;   // 2^120
    out = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&bits), *reinterpret_cast<const __nv_bfloat162*>(&up));
  } else {
    const uint32_t low = (x & 0x007f007fu) | 0x43004300u, off = (x & 0x00800080u) | 0x43004300u;
    out = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&low), *reinterpret_cast<const __nv_bfloat162*>(&off));
  }
  return *reinterpret_cast<uint32_t*>(&out);
}
// The selector for byte i of the first word, and byte j of it or (4 + j) of the second.
__device__ __forceinline__ constexpr uint32_t code_pick(int i, int j) { return static_cast<uint32_t>(i * 0x11 | j * 0x1100); }

__device__ __forceinline__ void quant_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// PARTS bfloat16 parts of a pair of float32 numbers, largest first.
template <int PARTS> __device__ __forceinline__ void split_pair(float x, float y, uint32_t (&out)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    __nv_bfloat162 part = __floats2bfloat162_rn(x, y);
    out[i] = *reinterpret_cast<uint32_t*>(&part);
    x -= __low2float(part);
    y -= __high2float(part);
  }
}

template <typename T> __device__ __forceinline__ float quant_exp2(float x) { return std::is_same<T, float>::value ? exp2f(x) : decode_exp2(x); }

// Blocks resident on an SM: what the ring leaves room for, less for the registers of float32's parts.
template <typename T, int HD> struct QuantBlocks {
  static constexpr int value = std::is_same<T, float>::value ? (HD == 256 ? 1 : 3) : (HD == 256 ? 2 : 4);
};

template <typename T, int KIND, int HD, bool BIASED>
__global__ void __launch_bounds__(kDecodeThreads, QuantBlocks<T, HD>::value)
quantized_decode_mma_kernel(const QuantizedDecode a) {
  using Tile = QuantTile<HD>;
  constexpr int PARTS = std::is_same<T, float>::value ? 3 : 1;
  constexpr int WARPS = kDecodeThreads / 32, STAGES = Tile::kStages, STEPS = HD / 16;
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

  // Stage i of the warp: half i & 1 of its keys of the block's tile i / 2.
  const int stages = 2 * ((walk.count - rank + slots - 1) / slots);
  auto first_of = [&](int i) { return walk.tile(rank + (i >> 1) * slots) * kSplitKeys + warp * 32 + (i & 1) * Tile::kKeys; };
  auto holds = [&](int key0) { return key0 <= pos && (key0 + Tile::kKeys > first_key || key0 < a.keep); };
  // The pool row of key `lane % 16` of stage i: negative where the token does not see it.
  auto row_of = [&](int i) {
    const int key = first_of(i) + (lane & 15);
    return i < stages && key_seen(key, pos, first_key, a.keep)
               ? quantized_row(table, a.max_pages, a.num_pages, a.kv_heads, kv, a.page_tokens, key, a.status) : -1;
  };
  const int value_rows = a.kv_heads * a.page_tokens;   // from a key's row to its value's
  auto issue = [&](int i, int own_row) {
    if (i < stages && holds(first_of(i))) {
      unsigned char* at = ring + (i % STAGES) * Tile::kStageBytes;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int r = __shfl_sync(0xffffffffu, own_row, b * 8 + g);
        const uint8_t* src = a.codes + static_cast<size_t>(max(r, 0)) * HD + t * 16;
#pragma unroll
        for (int j = 0; j < Tile::kKeyPieces; ++j)
          quant_copy<16>(at + ((b * Tile::kKeyPieces + j) * 32 + lane) * 16, src + j * 64, r >= 0);
      }
      at += Tile::kRowBytes;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int r = __shfl_sync(0xffffffffu, own_row, 2 * t + (n & 1) + (n >> 1) * 8);
        const uint8_t* src = a.codes + (static_cast<size_t>(max(r, 0)) + value_rows) * HD + g * Tile::kValueBytes;
#pragma unroll
        for (int j = 0; j < Tile::kValuePieces; ++j)
          quant_copy<Tile::kValueBytes>(at + ((n * Tile::kValuePieces + j) * 32 + lane) * Tile::kValueBytes, src + j * 128, r >= 0);
      }
      at += 4 * Tile::kValuePieces * Tile::kValueBytes * 32;
      quant_copy<4>(at + lane * 4, a.scales + static_cast<size_t>(max(own_row, 0)) + (lane < 16 ? 0 : value_rows), own_row >= 0);
    }
    asm volatile("cp.async.commit_group;\n" ::);
  };
  // The token's own row, of the walk's last tile, is written by the kernel ahead of this one; with `settled` all others
  // are older, and their copies start ahead of the wait.
  bool waited = !a.settled;
  int own_row = row_of(0);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (!waited && i < stages && first_of(i) + Tile::kKeys > pos) {
      chain_wait();
      waited = true;
    }
    const int next_row = row_of(i + 1);
    issue(i, own_row);
    own_row = next_row;
  }
  if (!waited) chain_wait();

  // ---- the query heads as rows 0..7 (float32: their second parts as rows 8..15, their third in a product of its own)
  uint32_t q0[STEPS][PARTS], q2[STEPS][PARTS];
  {
    const T* q = behind_wait(static_cast<const T*>(a.q)) + (static_cast<size_t>(token) * a.heads + head0 + (g < live ? g : 0)) * HD;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const T* at = q + (s >> 2) * 64 + t * 16 + (s & 3) * 4;
      alignas(16) T values[4];
      if (PARTS == 1) *reinterpret_cast<uint2*>(values) = *reinterpret_cast<const uint2*>(at);
      else *reinterpret_cast<uint4*>(values) = *reinterpret_cast<const uint4*>(at);
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = g < live ? to_float(values[i]) : 0.0f;
      split_pair<PARTS>(x[0], x[1], q0[s]);
      split_pair<PARTS>(x[2], x[3], q2[s]);
    }
  }
  float m_run = -INFINITY, l_run = 0.0f;   // of head g, over this warp's keys so far
  float o[HD / 16][4];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

  for (int i = 0; i < stages; ++i) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2));
    __syncwarp();   // every lane's copies of stage i have landed, and every lane is done with stage i - 1
    const int next_row = row_of(i + STAGES);
    issue(i + STAGES - 1, own_row);
    own_row = next_row;
    const int key0 = first_of(i);
    if (!holds(key0)) continue;
    const unsigned char* at = ring + (i % STAGES) * Tile::kStageBytes;
    const float* scales = reinterpret_cast<const float*>(at + Tile::kStageBytes - 2 * Tile::kKeys * 4);

    // ---- scores of 16 keys: this lane has those of head g and keys b * 8 + 2t, 2t + 1
    float s[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < Tile::kKeyPieces; ++j) {
        const uint4 piece = *reinterpret_cast<const uint4*>(at + ((b * Tile::kKeyPieces + j) * 32 + lane) * 16);
        const uint32_t words[4] = {piece.x, piece.y, piece.z, piece.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t b0 = code_pair<KIND>(words[w], words[w], code_pick(0, 1));
          const uint32_t b1 = code_pair<KIND>(words[w], words[w], code_pick(2, 3));
          const int n = j * 4 + w;
          if (PARTS == 1) {
            quant_mma(d, q0[n][0], 0u, q2[n][0], 0u, b0, b1);
          } else {
            quant_mma(d, q0[n][0], q0[n][PARTS - 2], q2[n][0], q2[n][PARTS - 2], b0, b1);
            quant_mma(d, q0[n][PARTS - 1], 0u, q2[n][PARTS - 1], 0u, b0, b1);
          }
        }
      }
      const float2 k_scale = *reinterpret_cast<const float2*>(scales + b * 8 + 2 * t);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = key0 + b * 8 + 2 * t + j;
        float score = capped_score((d[j] + d[2 + j]) * (j ? k_scale.y : k_scale.x) * a.scale, a.softcap);
        if (BIASED && g < live) score += bias_at(a.bias.row(head0 + g), pos - key, a.bias.far);
        s[b][j] = key_seen(key, pos, first_key, a.keep) ? score * kLog2E : -INFINITY;
      }
    }
    float m_new = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
    m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 1));
    m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 2));
    m_new = fmaxf(m_new, m_run);
    const float ref = m_new == -INFINITY ? 0.0f : m_new;
    const float carry = quant_exp2<T>(m_run - ref);   // what earlier stages gathered, on the new maximum (0 if nothing yet)
    const bool moved = __any_sync(0xffffffffu, m_new != m_run);
    float l_new = 0.0f;
    uint32_t p[2][PARTS];   // the weights of key pairs b * 8 + 2t, 2t + 1, times the values' scales
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float p0 = quant_exp2<T>(s[b][0] - ref), p1 = quant_exp2<T>(s[b][1] - ref);
      l_new += p0 + p1;
      const float2 v_scale = *reinterpret_cast<const float2*>(scales + Tile::kKeys + b * 8 + 2 * t);
      split_pair<PARTS>(p0 * v_scale.x, p1 * v_scale.y, p[b]);
    }
    l_run = l_run * carry + l_new;   // this lane's keys alone; the four lanes of a head meet at the end
    m_run = m_new;
    if (moved) {
      const float c0 = __shfl_sync(0xffffffffu, carry, 8 * t), c1 = __shfl_sync(0xffffffffu, carry, 8 * t + 4);   // heads 2t, 2t + 1
#pragma unroll
      for (int n = 0; n < HD / 16; ++n) { o[n][0] *= c0; o[n][1] *= c1; o[n][2] *= c0; o[n][3] *= c1; }
    }
    // ---- o^T += V^T p^T
    at += Tile::kRowBytes;
#pragma unroll
    for (int j = 0; j < Tile::kValuePieces; ++j) {
      constexpr int WORDS = Tile::kValueBytes / 4;
      uint32_t v[4][WORDS];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const unsigned char* src = at + ((n * Tile::kValuePieces + j) * 32 + lane) * Tile::kValueBytes;
        if (WORDS == 4) *reinterpret_cast<uint4*>(v[n]) = *reinterpret_cast<const uint4*>(src);
        else *reinterpret_cast<uint2*>(v[n]) = *reinterpret_cast<const uint2*>(src);
      }
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int i0 = 2 * half, i1 = 2 * half + 1;
          const uint32_t a0 = code_pair<KIND>(v[0][w], v[1][w], code_pick(i0, 4 + i0));
          const uint32_t a1 = code_pair<KIND>(v[0][w], v[1][w], code_pick(i1, 4 + i1));
          const uint32_t a2 = code_pair<KIND>(v[2][w], v[3][w], code_pick(i0, 4 + i0));
          const uint32_t a3 = code_pair<KIND>(v[2][w], v[3][w], code_pick(i1, 4 + i1));
#pragma unroll
          for (int x = 0; x < PARTS; ++x) quant_mma(o[j * 2 * WORDS + 2 * w + half], a0, a1, a2, a3, p[0][x], p[1][x]);
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
#pragma unroll
  for (int n = 0; n < HD / 16; ++n) {
    constexpr int BLOCKS = Tile::kValueBytes / 2;   // of 16 values, from one piece
    const int d = (n / BLOCKS) * 128 + g * Tile::kValueBytes + (n % BLOCKS) * 2;
    float* to = merge + (warp * 8 + 2 * t) * (HD + 2) + d;
    to[0] = o[n][0];
    to[1] = o[n][2];
    to[HD + 2] = o[n][1];
    to[HD + 3] = o[n][3];
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
      const float weight = exp2f(theirs[HD] - m_all);   // a warp without keys has m = -inf: weight 0
      sum += weight * theirs[d];
      l_all += weight * theirs[HD + 1];
    }
    float* dst = a.partial + ((static_cast<size_t>(row) * a.heads + head0 + h) * slots + rank) * (HD + 2);
    dst[d] = sum;
    if (d == 0) { dst[HD] = m_all * 0.6931471805599453f; dst[HD + 1] = l_all; }   // the merge kernel works in natural units
  }
}

// Whether the tensor-core kernel takes these rows: pieces of 16 bytes (queries: 8 or 16) that lie on such boundaries.
static bool quantized_mma_takes(const QuantizedDecode& a) {
  return (a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) && reinterpret_cast<uintptr_t>(a.codes) % 16 == 0 &&
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
