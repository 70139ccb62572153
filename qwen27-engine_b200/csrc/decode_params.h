// Parameters shared by the two split-K decode kernels (decode.cu: warp-MMA kernel; decode_tc.cu:
// tcgen05 kernel) and the launcher of the latter.
#pragma once
#include "host.h"

namespace q27b {

struct DecodeParams {
  const float* qn;   // [T][nqh][256]
  float* part;       // [nkvh][nch][24][258]
  const int* pos0;
  int* status;
  int T, nqh, nkvh, n_ctx, nch;
  float kq_scale;
  int base_pos;      // global position of local cache row 0
  int n_local;       // local rows to attend; < 0: all rows up to *pos0 + T
  // paged / batched variant: grid (chunks, nkvh, B), fixed chunk length, rows through the page table
  const int* page_table;  // [B][max_pages]
  const int* seq_len;     // [B], counts the T new tokens
  int max_pages, n_pages, chunk_len;
  // Tile pool of the warp-specialised kernel (one sequence only): [KV head] tiles drawn so far,
  // [32] CTAs that are done; all zero between launches. Null: every CTA keeps to its own share.
  int* sched;
  // measurement hook (null in normal use): [CTA][8] globaltimer stamps of the warp-specialised kernel
  unsigned long long* trace;
};

// Which rows the tokens of a decode kernel attend: up to their own (attn_decode), those before all of them (launch_prefix), or
// those of a list of blocks. The other two are kernels of their own, with their parameters apart: with a list's fields in
// DecodeParams and its code beside theirs, ptxas arranged the kernels of attn_decode otherwise, and they took longer (f16, 32,768
// positions, one and four tokens: 29.6 and 36.6 us a call without, 33.8 and 40.4 with; q8_0, 150,000, four: 76.8 and 81.6).
enum class Rows { ALL, PREFIX, LIST };
// Lists of blocks (T = 1, one "sequence" per (sequence, token)): [B][sel_T][nkvh][sel_k] 64-position blocks, -1 = none, chunk_len
// entries to a chunk; the partials go to part_o [row][nch][256] and part_ml [row][nch].
struct ListParams : DecodeParams {
  const int* sel;
  int sel_k, sel_T;
  float* part_o;
  float2* part_ml;
};
template <Rows ROWS> struct ParamsOf { using type = DecodeParams; };
template <> struct ParamsOf<Rows::LIST> { using type = ListParams; };

// One sequence: its tiles of 64 positions are dealt out to the nch chunks of a KV head in equal shares of up to
// ceil(tiles / nch) tiles; above this share the chunks keep back a common pool (decode_ws.cu) and every chunk has tiles.
constexpr int POOL_MIN_TILES = 8;
// How many of the nch partials of a KV head hold anything when n positions are attended (at least one: the first
// chunk's partial is always written).
__host__ __device__ inline int filled_chunks(int n, int nch) {
  const int tiles = (n + 63) / 64, share = (tiles + nch - 1) / nch;
  if (share > POOL_MIN_TILES) return nch;
  return tiles < 1 ? 1 : (tiles + share - 1) / share;
}

// Split-K decode over a q8_0 cache on the tcgen05 path (decode_tc.cu). Same grid, same partial
// layout and same tensor maps as the warp-MMA kernel. paged: rows through the page table.
int launch_decode_tc(const CUtensorMap* kv, const CUtensorMap* ks, const CUtensorMap* vv, const CUtensorMap* vs,
                     const DecodeParams& p, bool paged, int nseq, cudaStream_t s);

// The warp-specialised split-K kernel (decode_ws.cu): same grid, partial layout and tensor maps again.
// groups (paged launches only): PAIRED and SPREAD CTAs have 8 warps and one tile group instead of 16 warps and two; two
// PAIRED CTAs fit an SM, a SPREAD one has it to itself.
enum class WsGroups { TWO, PAIRED, SPREAD };
int launch_decode_ws(const CUtensorMap* kv, const CUtensorMap* ks, const CUtensorMap* vv, const CUtensorMap* vs,
                     const DecodeParams& p, bool paged, int nseq, cudaStream_t s, WsGroups groups = WsGroups::TWO);
// The same for the rows before the T tokens alone.
int launch_prefix_ws(const CUtensorMap* kv, const CUtensorMap* ks, const CUtensorMap* vv, const CUtensorMap* vs,
                     const DecodeParams& p, int nseq, cudaStream_t s);
int launch_prefix_ws_paged(const CUtensorMap* kv, const CUtensorMap* ks, const CUtensorMap* vv, const CUtensorMap* vs,
                           const DecodeParams& p, int nseq, cudaStream_t s, WsGroups groups);
// The same with the P V contraction on tcgen05 (decode_wt.cu).
int launch_decode_wt(const CUtensorMap* kv, const CUtensorMap* ks, const CUtensorMap* vv, const CUtensorMap* vs,
                     const DecodeParams& p, bool paged, int nseq, cudaStream_t s);
// Decode over lists of blocks: the warp-specialised kernel (q8_0, p.page_table null: contiguous; pairs: CTAs of one tile group,
// two to an SM, instead of two) and the single-role kernel of decode.cu (f16 caches). nseq = B * sel_T.
int launch_blocks_ws(const CUtensorMap* kv, const CUtensorMap* ks, const CUtensorMap* vv, const CUtensorMap* vs,
                     const ListParams& p, int nseq, cudaStream_t s, bool pairs);
int launch_blocks_f16(const CUtensorMap* kv, const CUtensorMap* vv, const ListParams& p, int nseq, cudaStream_t s);
// The attention of T = 1..4 tokens to the rows before them alone, by the kernels of a decode call (q8_0: the warp-specialised one;
// f16: decode.cu); partials [sequence][KV head][chunk][24][258].
struct PrefixPartials {
  const float* part;
  int nch;        // chunks of a KV head
  int chunk_len;  // their length over pages; 0: as filled_chunks says
};
int launch_prefix(DeviceCtx* ctx, const float* qn, const void* kcache, const void* vcache, const int* pos0, int T, float kq_scale,
                  int nkvh, int n_ctx, bool q8, PrefixPartials* out, cudaStream_t s);
int launch_prefix_paged(DeviceCtx* ctx, const float* qn, const void* kpool, const void* vpool, const int* page_table,
                        const int* seq_len, int B, int T, float kq_scale, int nkvh, int n_pages, int max_pages, int max_seq_len,
                        const char* who, PrefixPartials* out, cudaStream_t s);
// Opts the kernels of decode_ws.cu into their shared-memory size on the current device.
int decode_ws_setup();

}  // namespace q27b
