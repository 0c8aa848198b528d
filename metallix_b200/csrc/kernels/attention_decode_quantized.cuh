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

template <typename T>
static cudaError_t launch_quantized_decode(const QuantizedDecode& args, int kind, int rows, int slots, cudaStream_t stream) {
  const int parts = (args.heads / args.kv_heads + kQuantHeads - 1) / kQuantHeads;
  const dim3 grid(slots, args.kv_heads * parts, rows);
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

// How many blocks a (token, key/value head) pair gets: as many as fill the GPU
// with blocks resident at once, no more than it has tiles.
static int quantized_slots(int pairs, int max_splits) {
  const int wanted = pairs > 0 ? (kDecodeBlocksAtOnce + pairs - 1) / pairs : 1;
  return wanted < max_splits ? wanted : max_splits;
}

}  // namespace mxb
