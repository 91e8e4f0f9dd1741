// C ABI of beams and the states behind them (include/vsmp_beam.h): argument checks and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>

#include "vsmp_beam.hpp"
#include "vsmp_error.hpp"
#include "vsmp_internal.hpp"
#include "vsmp_logits.hpp"

namespace vsmp {
namespace {

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// -1 with the message set unless the planes are ones that the operators take.
int check_planes(const vsmp_planes& p) {
  if (!p.planes || !aligned(p.planes, 8)) return set_error("vsmp: planes must be a device array of addresses");
  if (p.n_planes < 1 || p.rows < 1 || p.pieces < 1 || p.tokens < 1 || p.token_bytes < 1)
    return set_error("vsmp: need at least one plane, row, piece, token and byte");
  const long long run = static_cast<long long>(p.tokens) * p.token_bytes;
  if (run > INT32_MAX || (run + 7) / 8 * p.pieces > INT32_MAX || p.n_planes > 1 << 20)
    return set_error("vsmp: a row's tokens must hold fewer than 2^31 bytes a piece and 2^34 in all, in at most 2^20 planes");
  const long long most = LLONG_MAX / 4;
  if (p.row_stride < 0 || p.row_stride > most / p.rows || (p.pieces > 1 && (p.piece_stride < 0 || p.piece_stride > most / p.pieces)))
    return set_error("vsmp: the planes' strides must be positive and the planes addressable");
  const long long row = p.pieces > 1 ? (p.pieces - 1) * p.piece_stride + run : run;
  const bool in_rows = (p.pieces == 1 || p.piece_stride >= run) && (p.rows == 1 || p.row_stride >= row);
  const bool in_pieces = (p.rows == 1 || p.row_stride >= run) && p.pieces > 1 && p.piece_stride >= (p.rows - 1) * p.row_stride + run;
  if (!in_rows && !in_pieces) return set_error("vsmp: the planes' rows and pieces overlap");
  return 0;
}

PlaneArgs plane_args(const vsmp_planes& p) {
  return {p.planes, p.n_planes, p.row_stride, p.pieces, p.pieces > 1 ? p.piece_stride : 0, p.tokens, p.token_bytes};
}

int check_pages(const vsmp_pages& p) {
  if (p.rows < 1 || p.rows > kPageRows) return set_error("vsmp: need 1 <= rows <= " + std::to_string(kPageRows));
  if (p.n_pages < 1 || p.n_pages > kPagesMax) return set_error("vsmp: need 1 <= n_pages <= " + std::to_string(kPagesMax));
  if (p.row_pages < 1 || p.page_tokens < 1 || static_cast<long long>(p.row_pages) * p.page_tokens > kPageRoom)
    return set_error("vsmp: need row_pages >= 1 and page_tokens >= 1, at most 2^30 tokens a row");
  if (!p.table || !p.lens || !p.ref || !aligned(p.table, 4) || !aligned(p.lens, 4) || !aligned(p.ref, 4))
    return set_error("vsmp: table, lens and ref are required, aligned to 4 bytes");
  if (p.ldt < p.row_pages || p.ldt > LLONG_MAX / 16 / p.rows) return set_error("vsmp: ldt must be >= row_pages and the table addressable");
  return 0;
}

// Whether n bytes at a and m bytes at b overlap.
bool overlap(const void* a, long long n, const void* b, long long m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + static_cast<uintptr_t>(m) && y < x + static_cast<uintptr_t>(n);
}

struct Span {
  const void* p;
  long long n;
};

int check_step(const vsmp_pages* from, const vsmp_pages* to, const vsmp_planes* cache) {
  if (!from || !to) return set_error("vsmp: from and to are required");
  if (check_pages(*from) != 0 || check_pages(*to) != 0) return -1;
  if (from->n_pages != to->n_pages || from->page_tokens != to->page_tokens)
    return set_error("vsmp: from and to must have the same pool: n_pages and page_tokens");
  if (to->row_pages < from->row_pages) return set_error("vsmp: to's rows must have room for from's: row_pages");
  const Span in[] = {{from->table, 4 * ((from->rows - 1) * from->ldt + from->row_pages)}, {from->lens, 4ll * from->rows}, {from->ref, 4ll * from->n_pages}};
  const Span out[] = {{to->table, 4 * ((to->rows - 1) * to->ldt + to->row_pages)}, {to->lens, 4ll * to->rows}, {to->ref, 4ll * to->n_pages}};
  for (const Span& o : out)
    for (const Span& i : in)
      if (overlap(i.p, i.n, o.p, o.n)) return set_error("vsmp: from and to must not overlap");
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < i; ++j)
      if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return set_error("vsmp: to's arrays must not overlap");
  if (cache) {
    if (check_planes(*cache) != 0) return -1;
    if (cache->rows != to->n_pages || cache->tokens != to->page_tokens)
      return set_error("vsmp: the cache's planes must have n_pages rows of page_tokens tokens");
    // copies are counted with 31 bits, a plane's 4 KB of a page each
    const long long cols = (static_cast<long long>(cache->tokens) * cache->token_bytes + 15) / 16 * cache->pieces;
    const long long chunks = (cols + kPageChunk - 1) / kPageChunk, pages = std::max(to->n_pages / 2 + 1, to->rows);
    if (chunks * cache->n_planes > INT32_MAX / pages)
      return set_error("vsmp: too many planes for so many pages: fewer than 2^31 pieces of 4 KB in half of the pool, or in a page of each row");
  }
  return 0;
}

}  // namespace
}  // namespace vsmp

extern "C" {

int vsmp_beam_select(vsmp_ctx* ctx, const void* logits, int dtype, long long ld, int G, int W, int V, const float* scores,
                     int N, const int* stop_ids, int n_stop, int* token, int* parent, float* score, int* end_token,
                     int* end_parent, float* end_score, int* n_end, void* stream) {
  using vsmp::aligned;
  using vsmp::set_error;
  vsmp::clear_error();
  if (!ctx) return set_error("vsmp: null context");
  if (!logits || !scores) return set_error("vsmp: logits and scores are required");
  if (dtype < VSMP_F32 || dtype > VSMP_F16) return set_error("vsmp: unknown dtype");
  if (G < 1 || W < 1 || V < 1 || N < 1) return set_error("vsmp: need G, W, V and N >= 1");
  if (W > vsmp::kBeamMax || N > vsmp::kBeamMax) return set_error("vsmp: at most " + std::to_string(vsmp::kBeamMax) + " beams a group");
  if (V > vsmp::kOpVocab) return set_error("vsmp: vocabulary larger than " + std::to_string(vsmp::kOpVocab));
  if (static_cast<long long>(G) * std::max(W, N) > INT32_MAX) return set_error("vsmp: more than 2^31 - 1 beams");
  if (ld < V || ld > (LLONG_MAX >> 4) / (static_cast<long long>(G) * W))
    return set_error("vsmp: the rows' stride must be >= V and the batch addressable");
  const size_t size = dtype == VSMP_F32 ? 4 : 2;
  if (!aligned(logits, size) || !aligned(scores, 4)) return set_error("vsmp: logits and scores must be aligned to their elements");
  if (n_stop < 0 || n_stop > vsmp::kBeamStops || (n_stop > 0 && !stop_ids))
    return set_error("vsmp: need 0 <= n_stop <= " + std::to_string(vsmp::kBeamStops) + " and the stop tokens");
  if (!token || !parent || !score) return set_error("vsmp: token, parent and score are required");
  if ((end_token == nullptr) != (end_parent == nullptr) || (end_token == nullptr) != (end_score == nullptr) ||
      (end_token == nullptr) != (n_end == nullptr))
    return set_error("vsmp: end_token, end_parent, end_score and n_end go together");
  for (const void* p : {static_cast<const void*>(token), static_cast<const void*>(parent), static_cast<const void*>(score),
                        static_cast<const void*>(end_token), static_cast<const void*>(end_parent), static_cast<const void*>(end_score),
                        static_cast<const void*>(n_end)})
    if (!aligned(p, 4)) return set_error("vsmp: outputs must be aligned to 4 bytes");
  vsmp::DeviceScope scope(vsmp::ctx_device(ctx));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!scope.ok() || !vsmp::stream_on_device(ctx, st)) return -1;
  vsmp::BeamArgs a{};
  if (!vsmp::beam_scratch(ctx, st, &a.s)) return -1;
  a.ld = ld;
  a.W = W;
  a.V = V;
  a.N = N;
  for (int i = 0; i < n_stop; ++i)  // those of the vocabulary, each once
    if (stop_ids[i] >= 0 && stop_ids[i] < V && std::find(a.stops, a.stops + a.n_stop, stop_ids[i]) == a.stops + a.n_stop)
      a.stops[a.n_stop++] = stop_ids[i];
  const int groups = std::max(1, vsmp::kBeamSlots / W);  // of one launch
  for (int g = 0; g < G; g += a.G) {
    a.G = std::min(groups, G - g);
    const long long row = static_cast<long long>(g) * W, out = static_cast<long long>(g) * N;
    a.row0 = static_cast<int>(row);
    a.x = static_cast<const char*>(logits) + row * ld * static_cast<long long>(size);
    a.scores = scores + row;
    a.token = token + out;
    a.parent = parent + out;
    a.score = score + out;
    if (end_token) {
      a.end_token = end_token + out;
      a.end_parent = end_parent + out;
      a.end_score = end_score + out;
      a.n_end = n_end + g;
    }
    vsmp::beam_parts(a.G * W, W, V, dtype, vsmp::ctx_cus(ctx), &a.P, &a.L);
    vsmp::launch_beam(a, dtype, st);
    if (!vsmp::hip_ok(hipGetLastError(), "beam launch")) return -1;
  }
  return 0;
}

int vsmp_reorder_rows(vsmp_ctx* ctx, const vsmp_planes* planes, const int* parent, int width, const int* len, void* stream) {
  using vsmp::set_error;
  vsmp::clear_error();
  if (!ctx) return set_error("vsmp: null context");
  if (!planes || !parent) return set_error("vsmp: planes and parent are required");
  if (vsmp::check_planes(*planes) != 0) return -1;
  if (width < 1 || width > vsmp::kBeamMax || planes->rows % width != 0)
    return set_error("vsmp: need 1 <= width <= " + std::to_string(vsmp::kBeamMax) + ", and rows in whole groups of it");
  if (!vsmp::aligned(parent, 4) || !vsmp::aligned(len, 4)) return set_error("vsmp: parent and len must be aligned to 4 bytes");
  vsmp::DeviceScope scope(vsmp::ctx_device(ctx));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!scope.ok() || !vsmp::stream_on_device(ctx, st)) return -1;
  vsmp::ReorderArgs a{};
  a.p = vsmp::plane_args(*planes);
  a.parent = parent;
  a.len = len;
  a.width = width;
  // a launch counts its columns of 8 bytes or more with 31 bits, its groups with 16
  const long long cols = (static_cast<long long>(planes->tokens) * planes->token_bytes + 7) / 8 * planes->pieces;
  const int most = static_cast<int>(std::min<long long>(planes->n_planes, INT32_MAX / cols)), groups = planes->rows / width;
  for (int g = 0, n; g < groups; g += n) {
    n = std::min(groups - g, 1 << 15);
    a.row0 = g * width;
    for (int p = 0; p < planes->n_planes; p += a.p.n_planes) {
      a.plane0 = p;
      a.p.n_planes = std::min(most, planes->n_planes - p);
      vsmp::launch_reorder(a, n, vsmp::ctx_cus(ctx), st);
      if (!vsmp::hip_ok(hipGetLastError(), "reorder launch")) return -1;
    }
  }
  return 0;
}

int vsmp_pages_step(vsmp_ctx* ctx, const vsmp_pages* from, const vsmp_pages* to, const int* parent, const int* add,
                    int add_all, const vsmp_planes* cache, int* ok, void* stream) {
  using vsmp::set_error;
  vsmp::clear_error();
  if (!ctx) return set_error("vsmp: null context");
  if (vsmp::check_step(from, to, cache) != 0) return -1;
  if (!vsmp::aligned(parent, 4) || !vsmp::aligned(add, 4) || !vsmp::aligned(ok, 4))
    return set_error("vsmp: parent, add and ok must be aligned to 4 bytes");
  vsmp::DeviceScope scope(vsmp::ctx_device(ctx));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!scope.ok() || !vsmp::stream_on_device(ctx, st)) return -1;
  vsmp::PageArgs a{};
  if (!vsmp::page_scratch(ctx, st, &a.s)) return -1;
  a.from = *from;
  a.to = *to;
  a.parent = parent;
  a.add = add;
  a.add_all = add_all;
  a.ok = ok;
  if (cache) a.cache = vsmp::plane_args(*cache);
  vsmp::launch_pages_step(a, vsmp::ctx_cus(ctx), st);
  return vsmp::hip_ok(hipGetLastError(), "pages launch") ? 0 : -1;
}

int vsmp_pages_compact(vsmp_ctx* ctx, const vsmp_pages* from, const vsmp_pages* to, const vsmp_planes* cache, int* moved,
                       int* live, void* stream) {
  using vsmp::set_error;
  vsmp::clear_error();
  if (!ctx) return set_error("vsmp: null context");
  if (vsmp::check_step(from, to, cache) != 0) return -1;
  if (from->rows != to->rows) return set_error("vsmp: from and to must have the same rows");
  if (!vsmp::aligned(moved, 4) || !vsmp::aligned(live, 4)) return set_error("vsmp: moved and live must be aligned to 4 bytes");
  vsmp::DeviceScope scope(vsmp::ctx_device(ctx));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!scope.ok() || !vsmp::stream_on_device(ctx, st)) return -1;
  vsmp::PageArgs a{};
  if (!vsmp::page_scratch(ctx, st, &a.s)) return -1;
  a.from = *from;
  a.to = *to;
  a.moved = moved;
  a.live = live;
  if (cache) a.cache = vsmp::plane_args(*cache);
  vsmp::launch_pages_compact(a, vsmp::ctx_cus(ctx), st);
  return vsmp::hip_ok(hipGetLastError(), "pages launch") ? 0 : -1;
}

}  // extern "C"
