// Paged 4-bit cache of keys and values: its layout, the lookup of a sequence's tokens in it and
// the parameters of the kernels that write, read and attend over it.
//
// Pool: [pages, kv_heads, page_size / 32, 40 d] bytes.  One unit of 40 d bytes holds K and V of 32
// consecutive tokens of one kv head (d = 64 or 128, G = d / 32 groups of 32 channels), so a
// reader fetches it with one bulk copy.  Every value is scale * code + low with a 4-bit code and
// fp16 scale and low per token and group (5 bits a value).  Inside a unit the bytes stand in the
// order in which a lane (g = lane / 4, t = lane % 4) of an m16n8k16 MMA needs them:
//   K codes   byte 0         token tau, 32-bit word t of group j (channels 32 j + 8 t + 0..7, lowest
//                            nibble first) at tau d/2 + 4 (t G + j): lane (g, t) reads the words
//                            of all groups of row tau = g as one 4 G-byte load
//   V codes   byte 16 d      tau = 16 blk + 8 h + 2 t + e, half-word (g, j) (channels 32 j + 4 g +
//                            0..3) at 8 d blk + 4 d h + 4 G (4 g + t) + 2 G e + 2 j: lane (g, t) reads
//                            its rows' channels for tokens 2t and 2t + 1 as one 4 G-byte load
//   K meta    byte 32 d      token tau: G scales, then G lows, at 4 G tau
//   V scales  + 128 G        at 32 G blk + 16 G h + 4 G t + 4 j + 2 e: half2 over tokens 2t, 2t + 1
//   V lows    + 64 G         the same
#pragma once
#include <cuda_fp16.h>

#include "kernels.cuh"

namespace rldx {

constexpr int kKv4Unit = 32;  // tokens of a unit and channels of a group

// Data errors of the cache kernels (record_data_error): an entry of the page table (or of lengths, cu_seqlens)
// names memory outside the pool, a RoPE row is outside its table, a sequence is longer or has
// more new tokens than the call said or a row to be stored belongs to none.  The access is skipped, the rest left out.
constexpr unsigned int kErrKv4Table = 0x500;
constexpr unsigned int kErrKv4Rope = 0x501;
constexpr unsigned int kErrKv4Bound = 0x502;
constexpr unsigned int kErrKv4Timeout = 0x510;

template <int D>
struct Kv4Unit {
  static constexpr int kG = D / 32;
  static constexpr int kBytes = 40 * D;
  static constexpr int kV = 16 * D;
  static constexpr int kKMeta = 32 * D;
  static constexpr int kVScale = kKMeta + 128 * kG;
  static constexpr int kVLow = kVScale + 64 * kG;
  static constexpr int kRow = D / 2;  // bytes of one token's codes
};

struct Kv4Cache {
  uint8_t* data;
  long long pages;
  int kv_heads, units_per_page;
  const int* table;  // [seqs, table_width], row stride table_ld
  int table_width, table_ld;
  const int* lengths;  // [seqs] tokens held, the new ones included
  const int* cu;       // [seqs + 1] rows of the new tokens
  int seqs, tokens;
};

// Index of unit `unit` (of sequence b, head h) in the pool, or -1 when the table names no page.  The
// host checks that a pool has fewer than 2^31 units.
__device__ __forceinline__ int kv4_unit_index(const Kv4Cache& c, int b, int h, int unit) {
  const int pg = unit / c.units_per_page;
  if (pg < 0 || pg >= c.table_width) return -1;
  const int id = __ldg(c.table + static_cast<long long>(b) * c.table_ld + pg);
  if (id < 0 || id >= c.pages) return -1;
  return (id * c.kv_heads + h) * c.units_per_page + (unit - pg * c.units_per_page);
}

struct Kv4AppendParams {
  Kv4Cache c;
  const __nv_bfloat16* qkv;  // [tokens, (Hq + 2 Hkv) d], row stride ld
  long long ld;
  int q_heads;
  const __nv_bfloat16* wq;
  const __nv_bfloat16* wk;
  const void* cos;  // [rope_rows, d] fp32 or bf16
  const void* sin;
  int rope_f32, rope_rows;
  const int* rope_pos;  // [tokens]
  __nv_bfloat16* q;     // [tokens, Hq, d]
  float eps;
};
cudaError_t launch_kv4_append(const Kv4AppendParams& p, int head_dim, cudaStream_t stream);

struct Kv4ReadParams {
  Kv4Cache c;
  __nv_bfloat16* k;  // [tokens, Hkv, d]
  __nv_bfloat16* v;
};
cudaError_t launch_kv4_read(const Kv4ReadParams& p, int head_dim, cudaStream_t stream);

struct Kv4AttnParams {
  Kv4Cache c;
  const __nv_bfloat16* q;  // [tokens, Hq, d], token stride ldq
  long long ldq;
  __nv_bfloat16* out;  // [tokens, Hq, d]
  int q_heads, group;
  int window, sinks;
  float scale_log2;
  int max_new, max_len;
  int whole;        // no segment is cut between CTAs
  float* part_o;    // [CTAs, 2, columns, d] unfinished results of a CTA's first and last segment
                    // (kv4_chunk_kernel: [CTAs, d / 4, 256, 4])
  float2* part_ml;  // [CTAs, 2, columns] their reference maximum (log2 units) and sum ([CTAs, 256])
  int4* part_head;  // [CTAs] first row, columns, kv head, parts and first CTA of the segment that a CTA begins,
                    // or (by_segment) of each segment: sequence, tile of columns, kv head
  int by_segment, tiles;
  int edges;           // this launch holds the batch's first sequence (1), its last (2)
  int split, ordered;  // kv4_chunk_kernel: CTAs that share the keys of a tile of rows; longest tiles first
};

// The units that the rows [row0, row0 + rows) of a sequence (row = new token * group + head of the
// group) can see: [0, sink_units) and [first, end), joined when they touch.
struct Kv4Span {
  int sink_units, first, end, count;
  int pos_lo, pos_hi;  // positions of the first and last row's tokens
  __device__ __forceinline__ int unit(int i) const { return i < sink_units ? i : first + i - sink_units; }
};

__device__ __forceinline__ Kv4Span kv4_span(int length, int nq, int tok_lo, int tok_hi, int window, int sinks) {
  Kv4Span s;
  s.pos_lo = length - nq + tok_lo;
  s.pos_hi = length - nq + tok_hi;
  const int keys = max(0, s.pos_hi + 1);
  s.end = (keys + kKv4Unit - 1) / kKv4Unit;
  s.first = window > 0 ? max(0, s.pos_lo - window + 1) / kKv4Unit : 0;
  s.first = min(s.first, s.end);
  s.sink_units = window > 0 ? (min(sinks, keys) + kKv4Unit - 1) / kKv4Unit : 0;
  if (s.first <= s.sink_units) s.first = s.sink_units = 0;
  s.count = s.sink_units + s.end - s.first;
  return s;
}

// Zeros in the output's rows [r0, r1), by thread i of n.
__device__ __forceinline__ void kv4_zero_rows(const Kv4AttnParams& P, int d, int r0, int r1, int i, int n) {
  const long long row = static_cast<long long>(P.q_heads) * d / 8;  // vectors of 16 bytes
  uint4* out = reinterpret_cast<uint4*>(P.out);
#pragma unroll 1
  for (long long at = max(r0, 0) * row + i; at < min(r1, P.c.tokens) * row; at += n) out[at] = make_uint4(0u, 0u, 0u, 0u);
}

cudaError_t launch_kv4_chunk(Kv4AttnParams p, int head_dim, cudaStream_t stream);
cudaError_t kv4_chunk_prepare_device();
cudaError_t launch_kv4_decode(const Kv4AttnParams& p, int head_dim, int cols, int warps, int ctas, int batch, cudaStream_t stream);

}  // namespace rldx
