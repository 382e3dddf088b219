// C ABI front end: argument checks, kernel selection, the host-side dense planner.
#include <algorithm>
#include <functional>
#include <queue>
#include <vector>

#include "common.cuh"
#include "nvtx_range.h"

namespace msa {
int fmha_mma_launch(const MsaFmhaParams& p, cudaStream_t stream);
int fmha_tc_supported(const MsaFmhaParams& p);
int fmha_tc_launch(const MsaFmhaParams& p, cudaStream_t stream);
int score_stream_supported(const MsaFmhaParams& p);
int score_stream_launch(const MsaFmhaParams& p, cudaStream_t stream);
int fmha_decode_tc_supported(const MsaFmhaParams& p);
int fmha_decode_tc_launch(const MsaFmhaParams& p, cudaStream_t stream);
int fmha_kv4_fwd(const MsaFmhaParams& p, cudaStream_t stream);
int fmha_window_supported(const MsaFmhaParams& p);
int fmha_window_launch(const MsaFmhaParams& p, cudaStream_t stream);
int fmha_sparse_tc_supported(const MsaFmhaParams& p);
int fmha_sparse_tc_launch(const MsaFmhaParams& p, cudaStream_t stream);
int64_t fmha_sparse_tc_workspace_bytes(int64_t total_q, int num_qo_heads, int num_kv_heads, int kbn, int64_t num_pages);
}  // namespace msa

namespace msa {
// Argument checks shared by every entry point that takes MsaFmhaParams.  Nothing here touches the
// device.  `own_scratch`: the split workspace is supplied by the library after this check
// (msa_fmha_fwd_split_static), so partial_o / partial_lse are expected to be NULL.
int validate_fmha(const MsaFmhaParams& p, bool own_scratch) {
  const bool sparse = (p.flags & MSA_FLAG_SPARSE) != 0;
  const bool has_o = (p.flags & MSA_FLAG_OUT_O) != 0;
  const bool has_s = (p.flags & MSA_FLAG_OUT_SCORE) != 0;
  if (!has_o && !has_s) return MSA_ERR_BAD_ARG;
  if (!p.q || !p.k || !p.qo_start || !p.kv_len || !p.qo_offset) return MSA_ERR_BAD_ARG;
  if (p.total_q < 0 || p.batch < 0) return MSA_ERR_BAD_ARG;
  if (has_o && (!p.v || (!p.out && !p.partial_o))) return MSA_ERR_BAD_ARG;
  if (has_s && (!p.max_score || p.max_k_tiles <= 0)) return MSA_ERR_BAD_ARG;
  if (own_scratch) {
    if (p.partial_o || p.partial_lse || p.num_splits < 1) return MSA_ERR_BAD_ARG;
  } else {
    if (p.partial_o && (!p.partial_lse || p.num_splits < 1)) return MSA_ERR_BAD_ARG;
    if (!p.partial_o && p.num_splits != 1) return MSA_ERR_BAD_ARG;
  }
  if (p.num_qo_heads <= 0 || p.num_kv_heads <= 0 || p.num_qo_heads % p.num_kv_heads) return MSA_ERR_BAD_ARG;
  const int h_r = p.num_qo_heads / p.num_kv_heads;
  if (p.pack < 1 || h_r % p.pack) return MSA_ERR_BAD_ARG;
  if (p.block_m != 16 && p.block_m != 64 && p.block_m != 128 && p.block_m != 256) return MSA_ERR_BAD_ARG;
  if (p.pack > p.block_m) return MSA_ERR_BAD_ARG;                 // rows of one token never straddle two items
  if (p.page_size > 0 && (!p.kv_page_indptr || !p.kv_indices)) return MSA_ERR_BAD_ARG;
  if (p.page_size <= 0 && !p.kv_start) return MSA_ERR_BAD_ARG;
  if (p.q_dtype != MSA_DT_BF16 && p.q_dtype != MSA_DT_E4M3) return MSA_ERR_UNSUPPORTED;
  if (p.kv_dtype != MSA_DT_BF16 && p.kv_dtype != MSA_DT_E4M3) return MSA_ERR_UNSUPPORTED;
  if (has_s && p.max_score_dtype != MSA_DT_F32 && p.max_score_dtype != MSA_DT_BF16) return MSA_ERR_UNSUPPORTED;
  if (p.window < 0 || p.sink_tokens < 0 || (p.sink_tokens > 0 && p.window == 0)) return MSA_ERR_BAD_ARG;
  if (p.window > 0 && (sparse || has_s)) return MSA_ERR_UNSUPPORTED;
  if (p.num_sms < 0) return MSA_ERR_BAD_ARG;
  if (sparse) {
    if (!p.kv_block_indexes || !p.token_batch || p.kv_block_num <= 0) return MSA_ERR_BAD_ARG;
    if (p.page_size != msa::kKvTile) return MSA_ERR_UNSUPPORTED;   // a selected block is one 128-key page
    if (has_s) return MSA_ERR_UNSUPPORTED;
    if (p.pack != h_r) return MSA_ERR_BAD_ARG;
  } else {
    if (p.num_work < 0 || (p.num_work > 0 && !p.work)) return MSA_ERR_BAD_ARG;
  }
  // 16-byte alignment of every row the kernels touch with vector accesses
  const int qe = p.q_dtype == MSA_DT_E4M3 ? 1 : 2, ke = p.kv_dtype == MSA_DT_E4M3 ? 1 : 2;
  auto al = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  if (!al(p.q) || !al(p.k) || (p.v && !al(p.v)) || (p.out && !al(p.out))) return MSA_ERR_BAD_ARG;
  if ((p.q_stride_tok * qe) % 16 || (p.q_stride_head * qe) % 16) return MSA_ERR_BAD_ARG;
  if ((p.k_stride_tok * ke) % 16 || (p.k_stride_head * ke) % 16 || (p.k_stride_page * ke) % 16) return MSA_ERR_BAD_ARG;
  if (has_o && ((p.v_stride_tok * ke) % 16 || (p.v_stride_head * ke) % 16 || (p.v_stride_page * ke) % 16)) return MSA_ERR_BAD_ARG;
  if (p.out && ((p.out_stride_tok * 2) % 16 || (p.out_stride_head * 2) % 16)) return MSA_ERR_BAD_ARG;
  return MSA_OK;
}
}  // namespace msa

extern "C" int msa_fmha_fwd(const MsaFmhaParams* pp, msa_stream_t stream_) {
  if (!pp) return MSA_ERR_BAD_ARG;
  msa::NvtxRange range("msa_fmha_fwd");
  const MsaFmhaParams& p = *pp;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (p.kv_dtype == MSA_DT_KV4) return msa::fmha_kv4_fwd(p, stream);
  if (const int rc = msa::validate_fmha(p, false)) return rc;
  if (msa::fmha_sparse_tc_supported(p)) return msa::fmha_sparse_tc_launch(p, stream);
  if (msa::score_stream_supported(p)) return msa::score_stream_launch(p, stream);
  if (msa::fmha_window_supported(p)) return msa::fmha_window_launch(p, stream);
  if (msa::fmha_decode_tc_supported(p)) return msa::fmha_decode_tc_launch(p, stream);
  if (msa::fmha_tc_supported(p)) return msa::fmha_tc_launch(p, stream);
  return msa::fmha_mma_launch(p, stream);
}

extern "C" int msa_fmha_fwd_merged(const MsaFmhaParams* pp, const int32_t* splits_per_row, int32_t out_dtype, msa_stream_t stream) {
  if (!pp || !pp->partial_o || !pp->partial_lse || !pp->out || pp->num_splits < 1) return MSA_ERR_BAD_ARG;
  if (out_dtype != MSA_DT_BF16 && out_dtype != MSA_DT_F32) return MSA_ERR_UNSUPPORTED;
  // all that the merge asks for, before anything is launched; `out` as in an unsplit call, rows that begin at multiples of 16 bytes
  const int oe = out_dtype == MSA_DT_BF16 ? 2 : 4;
  if ((reinterpret_cast<uintptr_t>(pp->partial_o) & 15) || (reinterpret_cast<uintptr_t>(pp->out) & 15) || pp->out_stride_tok * oe % 16 ||
      pp->out_stride_head * oe % 16)
    return MSA_ERR_BAD_ARG;
  if (static_cast<int64_t>(pp->total_q) * pp->num_qo_heads > 0x7fffffffLL) return MSA_ERR_TOO_LARGE;
  MsaFmhaParams p = *pp;
  p.out = nullptr;
  p.lse = nullptr;
  if (const int rc = msa_fmha_fwd(&p, stream)) return rc;
  return msa_lse_merge_many(p.partial_o, p.partial_lse, splits_per_row, pp->out, out_dtype, pp->lse, p.num_splits, p.total_q, p.num_qo_heads,
                            pp->out_stride_tok, pp->out_stride_head, p.out_scale, stream);
}

namespace msa {
struct Proto { int b, row0, nrows, ntiles, skip; };      // the rows of one work item and their KV tiles, before any split

// Tile times until the last of `slots` workers is done when every item is cut into pieces of `chunk` tiles and the
// pieces are handed out longest first.  A piece costs three tiles beyond its own (a CTA's dependent index loads, the
// latency of its first tile, its epilogue).
static int makespan(const std::vector<Proto>& protos, int groups, int chunk, int slots, int piece_cost = 3) {
  std::vector<int> pieces;
  for (const Proto& pr : protos)
    for (int t = pr.ntiles; t > 0; t -= chunk) pieces.push_back(std::min(t, chunk) + piece_cost);
  std::sort(pieces.begin(), pieces.end(), std::greater<int>());
  std::priority_queue<int, std::vector<int>, std::greater<int>> load(std::greater<int>(), std::vector<int>(slots, 0));
  int last = 0;
  for (const int t : pieces)
    for (int g = 0; g < groups; ++g) {
      const int end = load.top() + t;
      load.pop();
      load.push(end);
      last = std::max(last, end);
    }
  return last;
}

// Tiles of a piece of windowed decode.  Windows are short and alike, so that rounds of CTAs and the memory that all of them share decide.  In tile
// times of a CTA that nothing holds up (1.6 us in bf16, 16 rows; 1.4 times as much for more): a piece costs three beyond its own, a merge two and
// the partials' way to memory and back, memory gives each SM a tile in 0.9 (as if all were bf16), and of the two bounds a part of the
// smaller one shows as well.  Measured with 1 to 12 splits, merge included: 24 ragged sequences x 4 heads, at most 34 tiles: 60 us uncut, 40, 38
// (three), 43, 41 (seven), 47; 128 items of 10 tiles, 64 rows: 23, 24, 27 us; 512 of 66: 316, 326, 331 us; 512 of 18 e4m3 tiles: 61, 69, 73 us; one
// sequence of 10 tiles x 2 heads: 15.7, 11.7, 11.0, 8.3 us (five and ten).
//
// cluster > 1: a kernel whose CTAs share an uncut item, up to `cluster` of them with half a tile each at least, where all items are on the GPU at once
// (nine tenths of the places: a cluster stays within a group of SMs).  It needs no merge; joining the states takes half a tile's time.  Uncut so and
// cut: one sequence x 2 heads, 10 tiles 7.7 and 8.3 us; 16 x 2 x 9 tiles 9.4 and 10.3; 64 x 2 x 9 18.2 and 18.9; 32 x 2 x 33 28.1 and 29.2, but 4 x 2 x 33
// 11.3 and 9.8, and 48 x 2 x 33 e4m3 ones, of which two CTAs an item fit and not three, 34 and 29. The call is a launch and an allocation less on the
// host, 13 us instead of 18, for which such losses are taken.
static int window_chunk(const std::vector<Proto>& protos, int groups, int max_tiles, int slots, int sms, int ceiling, int cluster) {
  constexpr int kPieceCost = 3, kMerge = 2;
  long long total = 0, items = 0;
  for (const Proto& pr : protos) { total += static_cast<long long>(pr.ntiles) * groups; items += groups; }
  long long rows = 0;                                        // of partials, 0.5 KB each: 8 MB in a tile's time
  bool many = false;
  for (const Proto& pr : protos) { rows += static_cast<long long>(pr.nrows) * groups; many = many || pr.nrows > 16; }
  const double memory = 0.9 * static_cast<double>(total) / sms + kPieceCost, slow = many ? 1.4 : 1.0, merge_row = 1024 / 8e6;
  int best = std::max(1, max_tiles);
  if (items >= 8LL * slots) return best;
  double best_cost = 0;
  int last = 0;
  for (int s = 1; s <= std::min(max_tiles, ceiling); s += s < 8 ? 1 : s / 4) {
    const int chunk = (max_tiles + s - 1) / s;
    if (chunk == last || (s > 1 && items * s > 16LL * slots)) continue;
    last = chunk;
    const double ctas = slow * makespan(protos, groups, chunk, slots, kPieceCost);
    const double cost = std::max(memory, ctas) + 0.15 * std::min(memory, ctas) + (s > 1 ? kMerge + merge_row * s * rows : 0);
    if (s == 1 || cost < best_cost) { best = chunk; best_cost = cost; }
  }
  const long long share = std::min<long long>({cluster, 2LL * max_tiles, items > 0 ? slots * 9LL / 10 / items : 0});
  if (share > 1) {
    const double ctas = slow * (static_cast<double>(max_tiles) / share + kPieceCost + 0.5);
    if (std::max(memory, ctas) + 0.15 * std::min(memory, ctas) <= best_cost) best = std::max(1, max_tiles);
  }
  return best;
}
}  // namespace msa

extern "C" int msa_plan_dense(const MsaPlanArgs* a, MsaWorkItem* work, int32_t capacity, int32_t* splits_per_row,
                              int32_t* max_splits_out) {
  if (!a || !a->qo_len || !a->kv_len || !a->qo_offset || (!work && capacity > 0)) return MSA_ERR_BAD_ARG;
  msa::NvtxRange range("msa_plan_dense");
  if (a->block_m != 16 && a->block_m != 64 && a->block_m != 128 && a->block_m != 256) return MSA_ERR_BAD_ARG;
  if (a->num_qo_heads <= 0 || a->num_kv_heads <= 0 || a->num_qo_heads % a->num_kv_heads) return MSA_ERR_BAD_ARG;
  const int G = a->pack;
  if (G < 1 || (a->num_qo_heads / a->num_kv_heads) % G || G > a->block_m) return MSA_ERR_BAD_ARG;
  if (a->window < 0 || a->sink_tokens < 0 || (a->sink_tokens > 0 && a->window == 0)) return MSA_ERR_BAD_ARG;
  const int groups = a->num_qo_heads / G;
  const int bm_eff = (a->block_m / G) * G;       // a token's heads never straddle two items

  using msa::Proto;
  std::vector<Proto> protos;
  int max_tiles = 0;
  for (int b = 0; b < a->batch; ++b) {
    const int rows = a->qo_len[b] * G;
    for (int r0 = 0; r0 < rows; r0 += bm_eff) {
      const int nrows = std::min(bm_eff, rows - r0);
      const long long off = a->qo_offset[b];
      const msa::WindowSpan span = msa::window_span(r0 / G + off, (r0 + nrows - 1) / G + off, a->kv_len[b], a->window, a->sink_tokens);
      protos.push_back({b, r0, nrows, span.count, span.skip});
      max_tiles = std::max(max_tiles, span.count);
    }
  }
  // one chunk size (tiles per split) for the whole plan
  int chunk;
  if (a->num_splits >= 1) {
    chunk = std::max(1, (max_tiles + a->num_splits - 1) / a->num_splits);
  } else if (a->window > 0 && a->ctas_per_sm >= 0) {
    const int sms = a->num_sms > 0 ? a->num_sms : 148;
    chunk = msa::window_chunk(protos, groups, max_tiles, sms * std::max(1, a->ctas_per_sm), sms, a->num_splits < 0 ? -a->num_splits : 128, a->cluster);
  } else {
    const long long items = static_cast<long long>(protos.size()) * groups;
    const int ceiling = a->num_splits < 0 ? -a->num_splits : 128;
    const int sms = a->num_sms > 0 ? a->num_sms : 148;
    if (items == 0 || items >= 2LL * sms) {
      chunk = std::max(1, max_tiles);
    } else {
      int want = static_cast<int>((2LL * sms + items - 1) / items);
      want = std::min(want, ceiling);
      chunk = std::max(4, (max_tiles + want - 1) / want);      // at least 512 keys per split
    }
    // Decode: one row tile per batch item.  Cutting the items at just above the average load of an SM gives nearly every
    // SM one full piece and leaves the remainders to fill up the rest; whichever of the two cuts ends earlier is taken.
    // (Ragged lengths are where it pays: 31 sequences of 515 to 7 001 keys x 4 heads: 28 tile times against 40.)
    if (a->ctas_per_sm >= 0 && max_tiles > 4 && static_cast<int>(protos.size()) <= a->batch && items < 8LL * sms) {
      const int slots = sms * std::max(1, a->ctas_per_sm);
      long long total = 0;
      for (const Proto& pr : protos) total += static_cast<long long>(pr.ntiles) * groups;
      int cut = std::max(4, static_cast<int>((total * 103 + 100LL * slots - 1) / (100LL * slots)));
      // No more splits than the ceiling, nor than the library's own scratch holds where the plain cut fits it.  Every row
      // has as many partial rows as the longest item has splits, so one long sequence among many short ones would ask for
      // gigabytes: the partials take no more rows than those of a plain cut can (fewer than 2 x SMs items of block_m rows,
      // cut into 2 x SMs pieces or up to twice that), or what this batch's plain cut takes.
      long long rows = 0;
      for (int b = 0; b < a->batch; ++b) rows += static_cast<long long>(a->qo_len[b]) * a->num_qo_heads;
      rows = std::max(1LL, rows);
      const int plain_splits = (max_tiles + chunk - 1) / chunk;
      // (Three or more items to an SM: pieces so small that the cut they need has more rows, 0.5 KB each.  The kernel that runs
      // so has partials of its own call, and no form with the library's scratch.)
      const bool many = a->ctas_per_sm > 2;
      long long most = std::min<long long>(ceiling, std::max<long long>(plain_splits, (many ? 16LL * slots : 4LL * sms) * a->block_m / rows));
      if (!many && plain_splits * rows <= MSA_STATIC_SCRATCH_MAX_ROWS) most = std::min(most, MSA_STATIC_SCRATCH_MAX_ROWS / rows);
      cut = std::max(cut, static_cast<int>((max_tiles + most - 1) / most));
      if (cut < max_tiles && msa::makespan(protos, groups, cut, slots) < msa::makespan(protos, groups, chunk, slots)) chunk = cut;
    }
  }
  std::vector<MsaWorkItem> items;
  int max_splits = 1;
  std::vector<int> tok_base(a->batch + 1, 0);
  for (int b = 0; b < a->batch; ++b) tok_base[b + 1] = tok_base[b] + a->qo_len[b];
  for (const Proto& pr : protos) {
    const int ns = std::max(1, (pr.ntiles + chunk - 1) / chunk);
    max_splits = std::max(max_splits, ns);
    if (splits_per_row) {
      const int i0 = pr.row0 / G, i1 = (pr.row0 + pr.nrows - 1) / G;
      for (int i = i0; i <= i1; ++i) splits_per_row[tok_base[pr.b] + i] = ns;
    }
    for (int g = 0; g < groups; ++g)
      for (int s = 0; s < ns; ++s) {
        MsaWorkItem w;
        w.batch = pr.b; w.head0 = g * G; w.row0 = pr.row0;
        w.kv_tile_begin = std::min(pr.ntiles, s * chunk);
        w.kv_tile_end = std::min(pr.ntiles, (s + 1) * chunk);
        w.split = s; w.num_rows = pr.nrows; w.kv_tile_skip = pr.skip;
        items.push_back(w);
      }
  }
  std::stable_sort(items.begin(), items.end(), [](const MsaWorkItem& x, const MsaWorkItem& y) {
    return (x.kv_tile_end - x.kv_tile_begin) > (y.kv_tile_end - y.kv_tile_begin);
  });
  if (max_splits_out) *max_splits_out = max_splits;
  if (static_cast<long long>(items.size()) > capacity) return MSA_ERR_TOO_LARGE;
  std::copy(items.begin(), items.end(), work);
  return static_cast<int>(items.size());
}

extern "C" int64_t msa_sparse_workspace_bytes(int64_t total_q, int32_t num_qo_heads, int32_t num_kv_heads,
                                              int32_t kv_block_num, int64_t num_logical_pages) {
  if (total_q < 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || num_qo_heads % num_kv_heads || kv_block_num <= 0 ||
      num_logical_pages < 0)
    return MSA_ERR_BAD_ARG;
  return msa::fmha_sparse_tc_workspace_bytes(total_q, num_qo_heads, num_kv_heads, kv_block_num, num_logical_pages);
}

extern "C" const char* msa_status_string(int code) {
  switch (code) {
    case MSA_OK: return "ok";
    case MSA_ERR_BAD_ARG: return "bad argument (null pointer, misaligned or inconsistent sizes)";
    case MSA_ERR_UNSUPPORTED: return "unsupported combination of dtypes / modes / sizes";
    case MSA_ERR_LAUNCH: return "CUDA launch failed";
    case MSA_ERR_TOO_LARGE: return "size beyond a documented maximum";
    default: return "unknown status";
  }
}

extern "C" int msa_build_arch(void) { return 100; }

extern "C" int msa_sizeof(int which) {
  switch (which) {
    case 0: return static_cast<int>(sizeof(MsaFmhaParams));
    case 1: return static_cast<int>(sizeof(MsaWorkItem));
    case 2: return static_cast<int>(sizeof(MsaPlanArgs));
    case 3: return static_cast<int>(sizeof(MsaPlanDeviceArgs));
    case 4: return static_cast<int>(sizeof(MsaNormRopeArgs));
    case 5: return static_cast<int>(sizeof(MsaKv4ReadArgs));
    case 6: return static_cast<int>(sizeof(MsaPageTablesArgs));
    case 7: return static_cast<int>(sizeof(MsaPageCache));
    case 8: return static_cast<int>(sizeof(MsaPagesCopyArgs));
    case 9: return static_cast<int>(sizeof(MsaPagesForkArgs));
    case 10: return static_cast<int>(sizeof(MsaPagesFreeArgs));
    case 11: return static_cast<int>(sizeof(MsaPagesCompactArgs));
    default: return -1;
  }
}
