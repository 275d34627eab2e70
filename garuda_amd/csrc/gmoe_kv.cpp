// gmoe_kv.cpp — paged KV cache on the device and the decode-attention calls.
//
// The reference's KVCacheState (garuda/src/cache/mod.rs:221-600) holds one sequence's
// keys and values for one layer in blocks of `block_size` positions, capped at
// max_positions, with an optional sliding window (attention_start, :333-338). Here the
// blocks are pages of one device pool shared by every sequence and layer; the host keeps
// each (sequence, layer)'s length and page list, and the device keeps its page table,
// which the append kernel extends when a token opens a page. attend_one
// (llama/mod.rs:766-821) runs as one to five launches (gmoe_attn.hip). A cache may hold its
// complete blocks of 16 positions in 8 bits (gmoe_kv_create_q8, gmoe_attn8.hip).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <memory>
#include <mutex>
#include <new>
#include <stdexcept>
#include <vector>

#include "../../include/garuda_moe.h"
#include "gmoe_internal.h"

namespace gmoe {
void set_last_error(const char* msg);
int ctx_device(gmoe_ctx* c);
hipStream_t ctx_stream(gmoe_ctx* c);
}  // namespace gmoe

using namespace gmoe;

namespace {

gmoe_status kfail(gmoe_status s, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return s;
}

// The body of a C entry whose host planning allocates: no exception leaves it.
template <class F>
gmoe_status guarded(F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return kfail(GMOE_ERR_DEVICE, "no host memory for the call's plan");
  } catch (const std::length_error&) {
    return kfail(GMOE_ERR_DEVICE, "no host memory for the call's plan");
  }
}

#define KV_TRY(expr)                                                                       \
  do {                                                                                     \
    hipError_t e_ = (expr);                                                                \
    if (e_ != hipSuccess) return kfail(GMOE_ERR_DEVICE, "%s failed: %s", #expr, hipGetErrorString(e_)); \
  } while (0)

constexpr size_t kPinHalf = (size_t)512 << 10;  // bytes of a half at least
// a call has at most one tile per entry, and a place in the list of those in none
constexpr size_t kPinEntry = sizeof(AttnEntry) + sizeof(AttnTile) + sizeof(uint32_t);

struct Seq {
  bool open = false;
  std::vector<uint32_t> len;                 // [layer]
  std::vector<std::vector<uint32_t>> pages;  // [layer] page ids in position order
  std::vector<uint32_t> open_block;          // [layer] 8 bits: the block whose rows the open rows are
};

}  // namespace

struct gmoe_kv {
  gmoe_ctx* ctx = nullptr;
  gmoe_kv_desc d{};
  uint32_t kvd = 0, ppseq = 0;
  uint64_t page_floats = 0;
  float* pool = nullptr;      // [max_pages][2][block_size][kvd]; null in 8 bits
  bool q8 = false;            // complete blocks held in 8 bits
  Kv8Pool p8{};               // (with its tables and widths; a cache in f32 has only those)
  uint32_t* tables = nullptr; // [max_seqs][n_layers][ppseq]
  std::vector<uint32_t> free_pages;
  std::vector<Seq> seqs;
  uint8_t* scratch = nullptr; // per call: entries, rotated q, chunk partials
  size_t scratch_bytes = 0;
  uint32_t* done = nullptr;   // 8 bits: counters of written parts (Kv8Args), 0 between calls
  size_t n_done = 0;
  uintptr_t scratch_id = 0;   // another one whenever scratch or done moves
  // pinned staging of the entries and tiles of calls above kAttnInline tokens: two halves,
  // each taken from its start to its end; a half's event says its calls have read it
  uint8_t* pin = nullptr;
  size_t pin_half = 0, pin_at = 0;
  hipEvent_t pin_ev[2]{};
  int pin_cur = 0;
  float* saved = nullptr;      // 8 bits: a sequence's open rows, kept while a prompt runs (kv_snapshot)
  uint32_t fail_reserves = 0;  // test hook: reservations still to refuse (gmoe_kv_fail_reserves)
  std::mutex mu;

  ~gmoe_kv() {
    if (pool) hipFree(pool);
    if (tables) hipFree(tables);
    if (p8.codes) hipFree(p8.codes);
    if (p8.scales) hipFree(p8.scales);
    if (p8.open) hipFree(p8.open);
    if (p8.turns) hipFree(const_cast<double*>(p8.turns));
    if (saved) hipFree(saved);
    if (done) hipFree(done);
    if (scratch) hipFree(scratch);
    if (pin) hipHostFree(pin);
    for (auto& e : pin_ev)
      if (e) hipEventDestroy(e);
  }
};

namespace {

gmoe_status grow_scratch(gmoe_kv* kv, size_t bytes) {
  if (bytes <= kv->scratch_bytes) return GMOE_OK;
  KV_TRY(hipDeviceSynchronize());  // queued calls may still use the old buffer
  if (kv->scratch) KV_TRY(hipFree(kv->scratch));
  kv->scratch = nullptr;
  kv->scratch_bytes = 0;
  const size_t want = std::max(bytes, (size_t)8 << 20);
  kv->scratch_id++;
  KV_TRY(hipMalloc(&kv->scratch, want));
  kv->scratch_bytes = want;
  return GMOE_OK;
}

// Counters of n groups' parts a kv head.
gmoe_status grow_done(gmoe_kv* kv, size_t n) {
  n *= kv->d.n_kv_heads;
  if (n <= kv->n_done) return GMOE_OK;
  KV_TRY(hipDeviceSynchronize());  // queued calls may still use the old ones
  if (kv->done) KV_TRY(hipFree(kv->done));
  kv->done = nullptr;
  kv->n_done = 0;
  kv->scratch_id++;
  const size_t want = std::max(n, (size_t)4096);
  KV_TRY(hipMalloc((void**)&kv->done, want * sizeof(uint32_t)));
  KV_TRY(hipMemset(kv->done, 0, want * sizeof(uint32_t)));
  KV_TRY(hipDeviceSynchronize());  // before a call on any stream
  kv->n_done = want;
  return GMOE_OK;
}

// `bytes` of pinned memory for a call queued on st. An event is recorded, and waited for,
// once a half rather than once a call (5 us of idle GPU each). Calls on one cache are
// ordered on one stream, so the one that leaves a half records for all that used it.
gmoe_status take_pinned(gmoe_kv* kv, size_t bytes, hipStream_t st, uint8_t** out) {
  bytes = (bytes + 63) & ~(size_t)63;
  if (bytes > kv->pin_half) {
    if (kv->pin) {
      KV_TRY(hipDeviceSynchronize());  // queued calls may still read the old buffer
      KV_TRY(hipHostFree(kv->pin));
    }
    kv->pin = nullptr;
    kv->pin_half = kv->pin_at = 0;
    const size_t half = std::max(bytes, kPinHalf);
    KV_TRY(hipHostMalloc((void**)&kv->pin, 2 * half, hipHostMallocDefault));
    kv->pin_half = half;
  }
  if (kv->pin_at + bytes > kv->pin_half) {
    KV_TRY(hipEventRecord(kv->pin_ev[kv->pin_cur], st));
    kv->pin_cur ^= 1;
    kv->pin_at = 0;
    KV_TRY(hipEventSynchronize(kv->pin_ev[kv->pin_cur]));
  }
  *out = kv->pin + kv->pin_cur * kv->pin_half + kv->pin_at;
  kv->pin_at += bytes;
  return GMOE_OK;
}

// The call's entries (positions, windows, pages), checked against the window and the
// free pages but not committed; maxspan receives the longest span attended, distinct whether
// no two entries are of one sequence.
gmoe_status plan(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, AttnEntry* ent, uint32_t* maxspan,
                 bool* distinct = nullptr) {
  const gmoe_kv_desc& D = kv->d;
  if (layer >= D.n_layers) return kfail(GMOE_ERR_INFERENCE, "layer %u of %u", layer, D.n_layers);
  if (n == 0 || !seqs) return kfail(GMOE_ERR_INFERENCE, "empty attention call");
  std::vector<uint32_t> extra(kv->seqs.size(), 0);  // this call's entries so far, per sequence
  uint32_t need_pages = 0;
  *maxspan = 1;
  bool once = true;
  for (uint32_t i = 0; i < n; i++) {
    const uint32_t s = seqs[i];
    if (s >= kv->seqs.size() || !kv->seqs[s].open) return kfail(GMOE_ERR_INFERENCE, "sequence %u is not open", s);
    once &= extra[s] == 0;
    const uint32_t pos = kv->seqs[s].len[layer] + extra[s]++;
    if (pos >= D.max_positions)
      return kfail(GMOE_ERR_CACHE, "context window of %u positions is exhausted", D.max_positions);
    if (pos % D.block_size == 0) need_pages++;
    const uint32_t start = D.sliding_window && pos + 1 > D.sliding_window ? pos + 1 - D.sliding_window : 0;
    *maxspan = std::max(*maxspan, pos + 1 - start);
    ent[i].pos = pos;
    ent[i].start = start;
    ent[i].pages = kv->tables + ((size_t)s * D.n_layers + layer) * kv->ppseq;
  }
  if (need_pages > kv->free_pages.size())
    return kfail(GMOE_ERR_CACHE, "the KV pool has %zu free pages, the call needs %u", kv->free_pages.size(),
                 need_pages);
  if (distinct) *distinct = once;
  return GMOE_OK;
}

// Commits a planned call: lengths advance and pages are taken.
void commit(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, AttnEntry* ent) {
  const gmoe_kv_desc& D = kv->d;
  for (uint32_t i = 0; i < n; i++) {
    Seq& S = kv->seqs[seqs[i]];
    if (ent[i].pos % D.block_size == 0) {
      const uint32_t p = kv->free_pages.back();
      kv->free_pages.pop_back();
      S.pages[layer].push_back(p);
      ent[i].fresh = 1;
    } else {
      ent[i].fresh = 0;
    }
    ent[i].page = S.pages[layer][ent[i].pos / D.block_size];
    S.len[layer] = ent[i].pos + 1;
    S.open_block[layer] = ent[i].pos / kKv8Block;
  }
}

// Workgroups a tiled call is split into at least, keys permitting: a tile's keys are split over
// workgroups until the call has about one workgroup a CU, each split keeping at least two key
// tiles. The key tiles of a split:
constexpr uint32_t kAttnTileWgs = 256;
uint32_t split_key_tiles(const gmoe_kv* kv, size_t ntile, uint32_t span) {
  const uint32_t kt = (span + kAttnTileKeys - 1) / kAttnTileKeys;
  const uint32_t wgs = (uint32_t)ntile * kv->d.n_kv_heads;
  const uint32_t ns = std::max(1u, std::min((kAttnTileWgs + wgs - 1) / wgs, kt / 2));
  return (kt + ns - 1) / ns;
}

// How a call's entries are attended. Above kAttnInline tokens, runs (consecutive entries of one
// sequence: a prompt's positions) of at least an eighth of a tile of rows are cut into tiles of
// kAttnTileRows (token, query head) rows. Shorter runs leave the MFMA rows mostly empty: decode
// batches have no tiles, and beside a prompt such runs are singles, attended token by token in
// two more launches, unless as tiles of their own they leave every split with few keys. 32 heads
// on 8 of 128, 300 prompt tokens beside 30 sequences at 4000: all in tiles 630 us, singles apart
// 350, all token by token 874; 8 heads on 2 of 32, 64 tokens beside 3 sequences at 3000: 23, 33 and 30.
// span and chunks: the most keys a tile reads, and the most chunks of kAttnChunk a single attends.
struct Runs {
  std::vector<AttnTile> tiles;
  std::vector<uint32_t> singles;
  uint32_t span = 1, chunks = 1;
};
constexpr uint32_t kAttnFewKeyTiles = 4;
Runs find_runs(const gmoe_kv* kv, const AttnEntry* ent, uint32_t n, const float* out) {
  const uint32_t G = kv->d.n_heads / kv->d.n_kv_heads;
  // the tiles' rows are written 16 bytes at a time
  if (n <= kAttnInline || !attn_tiled_hd(kv->d.head_dim) || (uintptr_t)out % 16) return {};
  auto find = [&](bool short_too) {
    Runs R;
    for (uint32_t i = 0, j; i < n; i = j) {
      for (j = i + 1; j < n && ent[j].pages == ent[i].pages;) j++;
      const uint32_t rows = (j - i) * G;
      if (!short_too && 8 * rows < kAttnTileRows) {
        for (uint32_t k = i; k < j; k++) {
          R.singles.push_back(k);
          R.chunks = std::max(R.chunks, (ent[k].pos - ent[k].start) / kAttnChunk + 1);
        }
        continue;
      }
      for (uint32_t r = 0; r < rows; r += kAttnTileRows) {
        const uint32_t nr = std::min(kAttnTileRows, rows - r);
        const AttnEntry &f = ent[i + r / G], &e = ent[i + (r + nr - 1) / G];
        R.span = std::max(R.span, e.pos + 1 - f.start);
        R.tiles.push_back(AttnTile{i, r, nr, f.start, f.pos, e.start, e.pos, 0, f.pages});
      }
    }
    return R;
  };
  Runs R = find(false);
  if (R.singles.empty()) return R;
  // few tokens in tiles beside others are not worth two more launches
  if (n - R.singles.size() <= kAttnInline) return {};
  Runs all = find(true);
  return split_key_tiles(kv, all.tiles.size(), all.span) <= kAttnFewKeyTiles ? all : R;
}

// Scratch of a call of n entries and nchunk chunks: entries and tiles, rotated q, partials.
struct AttnLayout {
  size_t o_ent, o_qr, o_part, total;
};
AttnLayout layout(const gmoe_kv* kv, uint32_t n, uint32_t nchunk) {
  const gmoe_kv_desc& D = kv->d;
  const size_t qn = (size_t)n * D.n_heads * D.head_dim;
  AttnLayout l;
  l.o_ent = 0;
  l.o_qr = (n * kPinEntry + 255) & ~(size_t)255;
  l.o_part = l.o_qr + ((qn * 4 + 255) & ~(size_t)255);
  l.total = l.o_part + (size_t)n * D.n_heads * nchunk * (D.head_dim + 2) * 4;
  return l;
}

AttnArgs args(const gmoe_kv* kv, uint32_t n, uint32_t nchunk, const AttnLayout& l, const float* q, const float* k,
              const float* v, float* out, uint32_t q_stride, uint32_t kv_stride) {
  const gmoe_kv_desc& D = kv->d;
  AttnArgs a{};
  a.n = n;
  a.n_heads = D.n_heads;
  a.n_kv = D.n_kv_heads;
  a.hd = D.head_dim;
  a.bs = D.block_size;
  a.theta = D.rope_theta;
  a.scale = 1.0f / std::sqrt((float)D.head_dim);
  a.pool = kv->pool;
  a.page_floats = kv->page_floats;
  a.q = q;
  a.k = k;
  a.v = v;
  a.qr = reinterpret_cast<float*>(kv->scratch + l.o_qr);
  a.part = reinterpret_cast<float*>(kv->scratch + l.o_part);
  a.nchunk = nchunk;
  a.ctx = out;
  a.q_stride = q_stride ? q_stride : D.n_heads * D.head_dim;
  a.kv_stride = kv_stride ? kv_stride : kv->kvd;
  return a;
}

// The calls that read their plan's pinned memory, or that advance the host's lengths, cannot
// be replayed: a graph would run them again on the memory of later calls.
gmoe_status refuse_capture(hipStream_t st) {
  hipStreamCaptureStatus c = hipStreamCaptureStatusNone;
  KV_TRY(hipStreamIsCapturing(st, &c));
  if (c != hipStreamCaptureStatusNone)
    return kfail(GMOE_ERR_INFERENCE, "a call that plans on the host cannot be captured into a graph");
  return GMOE_OK;
}

Kv8Args args8(const gmoe_kv* kv, uint32_t n, const float* q, const float* k, const float* v, float* out,
              uint32_t q_stride, uint32_t kv_stride) {
  const gmoe_kv_desc& D = kv->d;
  Kv8Args a{};
  a.p = kv->p8;
  a.n = n;
  a.n_heads = D.n_heads;
  a.window = D.sliding_window;
  a.scale = 1.0f / std::sqrt((float)D.head_dim);
  a.q = q;
  a.k = k;
  a.v = v;
  a.ctx = out;
  a.q_stride = q_stride ? q_stride : D.n_heads * D.head_dim;
  a.kv_stride = kv_stride ? kv_stride : kv->kvd;
  a.done = kv->done;
  return a;
}

// A call on a cache in 8 bits: its runs (consecutive entries of one sequence; job not yet
// known), and of each sequence its tokens in the call, its first position and its first block's
// job. Checked against the window and the free pages as plan() checks entries, run by run.
struct Plan8 {
  struct Of {
    uint32_t count = 0, pos0 = 0, job = 0;
  };
  std::vector<Kv8Run> runs;
  std::vector<uint32_t> seq;  // [run]
  std::vector<Of> of;         // [sequence]
  uint32_t njob = 0;
  bool distinct = true;       // no sequence has two entries
};
gmoe_status plan8(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, Plan8& P) {
  const gmoe_kv_desc& D = kv->d;
  if (layer >= D.n_layers) return kfail(GMOE_ERR_INFERENCE, "layer %u of %u", layer, D.n_layers);
  if (n == 0 || !seqs) return kfail(GMOE_ERR_INFERENCE, "empty attention call");
  P.of.resize(kv->seqs.size());
  for (uint32_t i = 0; i < n; i++) {
    if (i && seqs[i] == seqs[i - 1]) {
      P.runs.back().n++;
      continue;
    }
    const uint32_t s = seqs[i];
    if (s >= kv->seqs.size() || !kv->seqs[s].open) return kfail(GMOE_ERR_INFERENCE, "sequence %u is not open", s);
    P.runs.push_back(Kv8Run{i, 1, 0, 0, s * D.n_layers + layer});
    P.seq.push_back(s);
  }
  uint64_t need = 0;
  for (size_t r = 0; r < P.runs.size(); r++) {
    Plan8::Of& o = P.of[P.seq[r]];
    Kv8Run& R = P.runs[r];
    if (!o.count) o.pos0 = kv->seqs[P.seq[r]].len[layer];
    R.pos0 = o.pos0 + o.count;
    const uint64_t end = (uint64_t)R.pos0 + R.n;
    if (end > D.max_positions) return kfail(GMOE_ERR_CACHE, "context window of %u positions is exhausted", D.max_positions);
    need += (end + D.block_size - 1) / D.block_size - ((uint64_t)R.pos0 + D.block_size - 1) / D.block_size;
    const uint32_t before = o.count ? (o.pos0 % kKv8Block + o.count + kKv8Block - 1) / kKv8Block : 0;
    o.count += R.n;
    P.njob += (o.pos0 % kKv8Block + o.count + kKv8Block - 1) / kKv8Block - before;
    P.distinct &= o.count == 1;
  }
  if (need > kv->free_pages.size())
    return kfail(GMOE_ERR_CACHE, "the KV pool has %zu free pages, the call needs %llu", kv->free_pages.size(),
                 (unsigned long long)need);
  for (size_t r = 0; r < P.runs.size(); r++) {  // what commit8 may not fail at
    std::vector<uint32_t>& pages = kv->seqs[P.seq[r]].pages[layer];
    const size_t most = ((uint64_t)P.runs[r].pos0 + P.runs[r].n + D.block_size - 1) / D.block_size;
    if (most > pages.capacity()) pages.reserve(std::max(most, 2 * pages.capacity()));
  }
  return GMOE_OK;
}

// Commits a planned call: lengths advance and pages are taken.
void commit8(gmoe_kv* kv, uint32_t layer, const Plan8& P) {
  for (size_t r = 0; r < P.runs.size(); r++) {
    Seq& S = kv->seqs[P.seq[r]];
    const uint32_t end = P.runs[r].pos0 + P.runs[r].n;
    while ((uint64_t)S.pages[layer].size() * kv->d.block_size < end) {
      S.pages[layer].push_back(kv->free_pages.back());
      kv->free_pages.pop_back();
    }
    S.len[layer] = end;
    S.open_block[layer] = (end - 1) / kKv8Block;
  }
}

// The blocks that a committed call appends to, those of one sequence in position order.
void fill_jobs(const gmoe_kv* kv, uint32_t layer, Plan8& P, Kv8Job* jobs) {
  const uint32_t bs = kv->d.block_size;
  uint32_t nj = 0;
  for (size_t r = 0; r < P.runs.size(); r++) {
    Plan8::Of& o = P.of[P.seq[r]];
    Kv8Run& R = P.runs[r];
    const uint32_t b0 = o.pos0 / kKv8Block, end = o.pos0 + o.count, nb = (end + kKv8Block - 1) / kKv8Block - b0;
    if (R.pos0 == o.pos0) {
      const std::vector<uint32_t>& pages = kv->seqs[P.seq[r]].pages[layer];
      o.job = nj;
      for (uint32_t b = 0; b < nb; b++) {
        Kv8Job& j = jobs[nj++];
        j = Kv8Job{};
        j.table = R.table;
        j.block = b0 + b;
        j.page = pages[j.block * kKv8Block / bs];
        j.r0 = b ? 0 : o.pos0 % kKv8Block;
        j.n = std::min(kKv8Block - j.r0, end - (j.block * kKv8Block + j.r0));
        j.flags = (b ? 0 : kKv8First) | (j.r0 + j.n == kKv8Block ? kKv8Whole : 0) |
                  (j.r0 == 0 && j.block * kKv8Block % bs == 0 ? kKv8Fresh : 0);
        j.last = o.job + nb - 1;
      }
    }
    R.job = o.job + R.pos0 / kKv8Block - b0;
    for (uint32_t t = 0; t < R.n; t++) {
      const uint32_t pos = R.pos0 + t;
      jobs[o.job + pos / kKv8Block - b0].ent[pos % kKv8Block] = R.i0 + t;
    }
  }
}

// The runs cut into groups (job: the run's index, for now) of at most 16 rows, or into tiles of
// at most kv8_tile_rows. A group reads the cache for itself, but a call of few groups has them all on
// the card at once, where a tile's waves without rows idle; so runs of enough rows go in tiles
// where as groups they would make more workgroups than the CUs hold (two each, of heads wider than 128
// one) three times over, of wide heads, whose tiles are smaller, twice. 32 heads on 8 of 128, in groups
// and in tiles: 32 tokens at 3008 (448 workgroups) 29 and 35 us, at 12000 (1600) 51 and 48; 16 tokens
// of each of 6 sequences at 3008 (1344) 48 and 52, 32 (2688) 73 and 57. 64 tokens at 2000, 8 heads on 2
// of 32 (160): 18 and 25. 8 heads of 256 on one: 256 tokens from 0 (256) 39 and 42, 128 at 3000 (512)
// 56 and 56, 64 at 12000 (832) 79 and 70.
// Enough rows, of a run alone in its tile: what a step of a tile costs beside its products does not
// shrink with the rows, nor with the heads. 30 sequences at 3008: 48 and 64 rows of 128 131 and 160, 167
// and 163; 80 and 96 of 64 216 and 244, 259 and 255; 63 and 96 of 80 87 and 95, 129 and 97; 128 of 32
// 41 and 46; 56 of 256 76 and 62.
constexpr uint32_t kv8_tile_min(uint32_t hd) { return 32 + 4096 / kv8_width(hd); }
constexpr uint32_t kv8_group_wgs(uint32_t hd) { return hd <= 128 ? 1536 : 512; }
void cut_runs(const gmoe_kv* kv, const std::vector<Kv8Run>& runs, std::vector<Kv8Run>& groups, std::vector<Kv8Run>& tiles) {
  const uint32_t G = kv->d.n_heads / kv->d.n_kv_heads, T = kv8_group_tokens(G), w = kv->d.sliding_window;
  auto large = [&](const Kv8Run& r) { return (uint64_t)r.n * G >= kv8_tile_min(kv->d.head_dim); };
  uint64_t wgs = 0;
  for (const Kv8Run& r : runs)
    if (large(r)) {
      const uint32_t end = r.pos0 + r.n - 1;
      wgs += (uint64_t)((r.n + T - 1) / T) * kv8_parts_of(end, w && end + 1 > w ? end + 1 - w : 0) * kv->d.n_kv_heads;
    }
  for (uint32_t i = 0; i < runs.size(); i++) {
    const Kv8Run& r = runs[i];
    const bool tile = wgs > kv8_group_wgs(kv->d.head_dim) && large(r);
    for (uint32_t at = 0, m; at < r.n; at += m) {
      const uint32_t pos = r.pos0 + at;
      m = std::min(r.n - at, tile ? kv8_tile_rows(kv->d.head_dim) / G : std::min(T, kKv8Block - pos % kKv8Block));
      (tile ? tiles : groups).push_back(Kv8Run{r.i0 + at, m, pos, i, r.table});
    }
  }
}

// Positions of a tile's split, at least two steps of 64. Where a CU each leaves room for four splits
// or more, as many as there are CUs, but for one kept for the own blocks, which then have a split of their
// own: a split of few positions takes as long again for them (256 tokens at 1280, 32 heads on 8 of
// 128: 6 splits, the own blocks in the first, 52 us; in a seventh 47). Otherwise the number under which
// the call would end first, counted in steps: a workgroup's start and end take two, the own blocks
// one and a half for each 32 positions, the sums of 32 workgroups written and joined one. (Rounded up
// to a workgroup a CU at least, a second round is mostly empty: 600 tokens at 4000 in 4 splits 163 us, in 3
// 125; 4 times 300 at 3000 in 2 230, in 1 196 to 209.)
constexpr uint32_t kKv8TileWgs = 256;
uint32_t tile_split(const gmoe_kv* kv, const std::vector<Kv8Run>& tiles, uint32_t* splits, uint32_t* own) {
  uint32_t span = 1;
  for (const Kv8Run& t : tiles) {
    const uint32_t w = kv->d.sliding_window, from = w && t.pos0 + 1 > w ? t.pos0 + 1 - w : 0;
    span = std::max(span, (t.pos0 + t.n - 1) / kKv8Block * kKv8Block - std::min(t.pos0, from) / kKv8Block * kKv8Block);
  }
  const uint32_t steps = (span + 63) / 64, wgs = (uint32_t)tiles.size() * kv->d.n_kv_heads;
  uint32_t ns = kKv8TileWgs / wgs - 1;
  if (kKv8TileWgs / wgs < 4) {
    const uint32_t own_steps = 3 * (kv8_tile_rows(kv->d.head_dim) / (kv->d.n_heads / kv->d.n_kv_heads) + 16) / 64;
    auto cost = [&](uint32_t n) -> uint64_t {
      const uint64_t each = (steps + n - 1) / n + 2, first = each + own_steps, left = (uint64_t)wgs * (n - 1);
      // the first splits start first: then `late` CUs are free at t1, the others at t0
      const uint64_t late = wgs % kKv8TileWgs, t0 = wgs / kKv8TileWgs * first, t1 = late ? t0 + first : t0;
      auto done = [&](uint64_t t) {  // of the others by then
        return (kKv8TileWgs - late) * ((t - t0) / each) + (t > t1 ? late * ((t - t1) / each) : 0);
      };
      uint64_t end = t1;
      if (left) {
        uint64_t a = t0, b = t1;
        while (done(a) < left) a += each;
        while (done(b) < left) b += each;
        end = std::max(t1, std::min(a, b));
      }
      return end + (n > 1 ? (uint64_t)wgs * n / 32 : 0);
    };
    ns = 1;
    for (uint32_t n = 2; n <= 8; n++)
      if (cost(n) < cost(ns)) ns = n;
  }
  ns = std::max(1u, std::min(ns, steps / 2));
  const uint32_t keys = (steps + ns - 1) / ns * 64;
  *splits = (span + keys - 1) / keys;
  *own = *splits > 1 && wgs * (*splits + 1) <= kKv8TileWgs ? 1 : 0;
  *splits += *own;
  return keys;
}

// Scratch of the partial sums of nx groups (tiles) of R rows a kv head.
size_t part8_bytes(const gmoe_kv* kv, size_t nx, uint32_t R, uint32_t nparts) {
  return (nparts * nx * kv->d.n_kv_heads * R * (kv->d.head_dim + 2) * 4 + 255) & ~(size_t)255;
}
size_t step8_bytes(const gmoe_kv* kv, uint32_t n, uint32_t nparts) {
  return part8_bytes(kv, n, kv->d.n_heads / kv->d.n_kv_heads, nparts);
}

// Whether a step's workgroups may write its context while others have yet to read: it lies
// apart from the inputs, or is the queries' own rows, which only a row's own workgroups read.
bool apart(const Kv8Args& a) {
  const size_t n = a.n, qd = (size_t)a.n_heads * a.p.hd, kvd = (size_t)a.p.n_kv * a.p.hd;
  auto over = [&](const float* p, size_t width, size_t stride) {
    const uintptr_t c = (uintptr_t)a.ctx, i = (uintptr_t)p;
    return c < i + ((n - 1) * stride + width) * 4 && i < c + n * qd * 4;
  };
  if (over(a.k, kvd, a.kv_stride) || over(a.v, kvd, a.kv_stride)) return false;
  return !over(a.q, qd, a.q_stride) || (a.ctx == a.q && a.q_stride == qd);
}

gmoe_status too_many(uint32_t n) { return kfail(GMOE_ERR_INFERENCE, "%u tokens are more than one launch takes", n); }

// attend() for a cache in 8 bits; with `out` null the tokens are only appended.
gmoe_status attend8(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, const float* q, const float* k,
                    const float* v, float* out, hipStream_t st, uint32_t q_stride, uint32_t kv_stride) {
  if (gmoe_status s = refuse_capture(st)) return s;
  Plan8 P;
  if (gmoe_status s = plan8(kv, layer, seqs, n, P)) return s;
  if (out)
    if (gmoe_status s = grow_done(kv, n)) return s;  // a group is of a token at least
  Kv8Args a = args8(kv, n, q, k, v, out, q_stride, kv_stride);
  const gmoe_kv_desc& D = kv->d;
  const uint32_t G = D.n_heads / D.n_kv_heads;
  auto start_of = [&](uint32_t pos) { return D.sliding_window && pos + 1 > D.sliding_window ? pos + 1 - D.sliding_window : 0; };
  uint8_t* pin = nullptr;
  if (out && P.distinct && apart(a)) {
    uint32_t span = 1;
    for (const Kv8Run& r : P.runs) {
      span = std::max(span, r.pos0 + 1 - start_of(r.pos0));
      a.items += kv8_parts_of(r.pos0, start_of(r.pos0));
    }
    a.nparts = kv8_parts(span);
    a.fused = kv8_fused(a.items, D.n_kv_heads, a.nparts, G * D.head_dim);
    if (!kv8_fits(a, true)) return too_many(n);
    const size_t eb = n > kKv8Inline ? (n * sizeof(AttnEntry) + 255) & ~(size_t)255 : 0;
    if (gmoe_status s = grow_scratch(kv, eb + step8_bytes(kv, n, a.nparts))) return s;
    if (eb)
      if (gmoe_status s = take_pinned(kv, eb, st, &pin)) return s;
    a.part = reinterpret_cast<float*>(kv->scratch + eb);
    commit8(kv, layer, P);
    Kv8Inline inl;
    AttnEntry* ent = pin ? reinterpret_cast<AttnEntry*>(pin) : inl.e;
    for (uint32_t i = 0; i < n; i++) {
      const uint32_t pos = P.runs[i].pos0;
      ent[i] = AttnEntry{kv->tables + (size_t)P.runs[i].table * kv->ppseq, pos, start_of(pos),
                         kv->seqs[P.seq[i]].pages[layer][pos / D.block_size], pos % D.block_size == 0 ? 1u : 0u};
    }
    if (pin) {
      KV_TRY(hipMemcpyAsync(kv->scratch, pin, n * sizeof(AttnEntry), hipMemcpyHostToDevice, st));
      a.ent = reinterpret_cast<const AttnEntry*>(kv->scratch);
    }
    KV_TRY(launch_kv8_step(a, inl, st));
    return GMOE_OK;
  }
  std::vector<Kv8Run> groups, tiles;
  size_t at = 0;
  auto take = [&](size_t bytes) {  // of the scratch
    const size_t o = at;
    at += (bytes + 255) & ~(size_t)255;
    return o;
  };
  a.njob = P.njob;
  if (!kv8_fits(a, false)) return too_many(n);
  size_t o_run = 0, o_qr = 0, o_own = 0, o_max = 0, o_part = 0, o_tpart = 0;
  if (out) {
    cut_runs(kv, P.runs, groups, tiles);
    a.nrun = (uint32_t)groups.size();
    a.ntile = (uint32_t)tiles.size();
    if (a.ntile) a.tkeys = tile_split(kv, tiles, &a.tsplits, &a.town);
    if (a.nrun) {
      uint32_t span = 1;
      for (const Kv8Run& g : groups) {
        span = std::max(span, g.pos0 + g.n - start_of(g.pos0));
        a.items += kv8_parts_of(g.pos0, start_of(g.pos0));
      }
      a.nparts = kv8_parts(span);
      a.fused = kv8_fused(a.items, D.n_kv_heads, a.nparts, kv8_group_tokens(G) * G * D.head_dim);
    }
    if (!kv8_fits(a, false)) return too_many(n);  // its groups and tiles
    o_run = take((groups.size() + tiles.size()) * sizeof(Kv8Run));
    o_qr = take((size_t)n * D.n_heads * D.head_dim * 4);
    o_own = take((size_t)P.njob * 2 * kKv8Block * kv->kvd * 4);
    o_max = take((size_t)P.njob * D.n_kv_heads * sizeof(float2));
    o_part = take(part8_bytes(kv, groups.size(), kv8_group_tokens(G) * G, a.nparts));
    o_tpart = take(part8_bytes(kv, tiles.size(), kv8_tile_rows(D.head_dim), a.tsplits));
    if (gmoe_status s = grow_scratch(kv, at)) return s;
  }
  const size_t jb = P.njob * sizeof(Kv8Job), rb = (groups.size() + tiles.size()) * sizeof(Kv8Run);
  Kv8CallInline inl;
  Kv8Job* jobs = inl.j;
  Kv8Run* runs = inl.r;
  if (P.njob > kKv8InlineJobs || groups.size() + tiles.size() > kKv8InlineRuns) {
    if (gmoe_status s = take_pinned(kv, jb + rb, st, &pin)) return s;
    a.hjob = jobs = reinterpret_cast<Kv8Job*>(pin);
    a.hrun = runs = reinterpret_cast<Kv8Run*>(pin + jb);
  }
  commit8(kv, layer, P);
  fill_jobs(kv, layer, P, jobs);
  for (const std::vector<Kv8Run>* v : {&groups, &tiles})
    for (Kv8Run r : *v) {  // a piece of run r.job
      const Kv8Run& of = P.runs[r.job];
      r.job = of.job + r.pos0 / kKv8Block - of.pos0 / kKv8Block;
      *runs++ = r;
    }
  if (out) {
    a.run = reinterpret_cast<Kv8Run*>(kv->scratch + o_run);
    a.qr = reinterpret_cast<float*>(kv->scratch + o_qr);
    a.own = reinterpret_cast<float*>(kv->scratch + o_own);
    a.own_max = reinterpret_cast<float2*>(kv->scratch + o_max);
    a.part = reinterpret_cast<float*>(kv->scratch + o_part);
    a.tpart = reinterpret_cast<float*>(kv->scratch + o_tpart);
  }
  KV_TRY(launch_kv8_call(a, inl, st));
  return GMOE_OK;
}

// The call's keys and values appended.
gmoe_status append(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, const float* k, const float* v,
                   hipStream_t st) {
  if (kv->q8) return attend8(kv, layer, seqs, n, nullptr, k, v, nullptr, st, 0, 0);
  if (gmoe_status s = refuse_capture(st)) return s;
  if (n > kMaxWgs) return too_many(n);
  std::vector<AttnEntry> ent(n ? n : 1);
  uint32_t maxspan;
  if (gmoe_status s = plan(kv, layer, seqs, n, ent.data(), &maxspan)) return s;
  AttnArgs a = args(kv, n, 0, AttnLayout{}, nullptr, k, v, nullptr, 0, 0);
  a.n_heads = 0;  // no queries
  uint8_t* pin = nullptr;
  if (n > kAttnInline)
    if (gmoe_status s = take_pinned(kv, n * sizeof(AttnEntry), st, &pin)) return s;
  commit(kv, layer, seqs, n, ent.data());
  if (pin) {
    memcpy(pin, ent.data(), n * sizeof(AttnEntry));
    a.ent = reinterpret_cast<const AttnEntry*>(pin);
  } else {
    std::copy(ent.begin(), ent.begin() + n, a.inl);
  }
  KV_TRY(launch_append(a, st));
  return GMOE_OK;
}

// The rows at positions pos[i] of seqs[i], in pieces of a block (in f32: of a page).
gmoe_status read_rows(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, const uint32_t* pos, uint32_t n, float* k,
                      float* v, hipStream_t st) {
  const gmoe_kv_desc& D = kv->d;
  if (layer >= D.n_layers) return kfail(GMOE_ERR_INFERENCE, "layer %u of %u", layer, D.n_layers);
  if (n == 0 || !seqs || !pos) return kfail(GMOE_ERR_INFERENCE, "empty read");
  if (gmoe_status s = refuse_capture(st)) return s;
  std::vector<Kv8Rows> rows;
  const uint32_t per = kv->q8 ? kKv8Block : D.block_size;
  uint32_t more = 0;  // positions that the last piece may still take: up to its end, or the sequence's
  for (uint32_t i = 0; i < n; i++) {
    const uint32_t s = seqs[i];
    if (more && s == seqs[i - 1] && pos[i] == pos[i - 1] + 1) {
      rows.back().n++;
      more--;
      continue;
    }
    if (s >= kv->seqs.size() || !kv->seqs[s].open) return kfail(GMOE_ERR_INFERENCE, "sequence %u is not open", s);
    const uint32_t len = kv->seqs[s].len[layer], b = pos[i] / per, r = pos[i] % per;
    if (pos[i] >= len) return kfail(GMOE_ERR_INFERENCE, "position %u of a sequence of %u", pos[i], len);
    rows.push_back(Kv8Rows{s * D.n_layers + layer, b, i, r, 1, kv->q8 && (uint64_t)(b + 1) * kKv8Block <= len});
    more = std::min(std::min(per - r, kKv8Block), len - pos[i]) - 1;
  }
  if (rows.size() * D.n_kv_heads > kMaxWgs) return too_many(n);
  Kv8RowsInline inl{};
  uint8_t* pin = nullptr;
  const size_t bytes = rows.size() * sizeof(Kv8Rows);
  if (rows.size() > kKv8Inline) {
    if (gmoe_status s = take_pinned(kv, bytes, st, &pin)) return s;
    memcpy(pin, rows.data(), bytes);
  } else {
    std::copy(rows.begin(), rows.end(), inl.r);
  }
  const Kv8Rows* list = reinterpret_cast<const Kv8Rows*>(pin);
  if (kv->q8) KV_TRY(launch_kv8_read(kv->p8, list, inl, (uint32_t)rows.size(), k, v, st));
  else KV_TRY(launch_kv_read(kv->p8, kv->pool, list, inl, (uint32_t)rows.size(), k, v, st));
  return GMOE_OK;
}

// Sequence s goes back to at most len positions in `layer`: pages past them are free again.
// Returns whether its open rows have to be made again from codes.
bool take_back(gmoe_kv* kv, uint32_t s, uint32_t layer, uint32_t len, Kv8Rows* rows) {
  Seq& S = kv->seqs[s];
  if (S.len[layer] <= len) return false;
  S.len[layer] = len;
  const uint32_t keep = (uint32_t)(((uint64_t)len + kv->d.block_size - 1) / kv->d.block_size);
  while (S.pages[layer].size() > keep) {
    kv->free_pages.push_back(S.pages[layer].back());
    S.pages[layer].pop_back();
  }
  const uint32_t b = len / kKv8Block;
  if (!kv->q8 || len % kKv8Block == 0 || S.open_block[layer] == b) return false;
  S.open_block[layer] = b;
  *rows = Kv8Rows{s * kv->d.n_layers + layer, b, 0, 0, len % kKv8Block, 1};
  return true;
}

gmoe_status truncate(gmoe_kv* kv, const uint32_t* seqs, const uint32_t* lens, uint32_t n, hipStream_t st) {
  if (n == 0 || !seqs || !lens) return kfail(GMOE_ERR_INFERENCE, "no sequences or lengths");
  if (gmoe_status s = refuse_capture(st)) return s;
  for (uint32_t i = 0; i < n; i++)
    if (seqs[i] >= kv->seqs.size() || !kv->seqs[seqs[i]].open)
      return kfail(GMOE_ERR_INFERENCE, "sequence %u is not open", seqs[i]);
  Kv8RowsInline inl{};
  uint32_t m = 0;
  for (uint32_t i = 0; i < n; i++) {
    // named before: its earlier rows may be waiting in inl
    if (m)
      for (uint32_t j = 0; j < i; j++)
        if (seqs[j] == seqs[i]) {
          KV_TRY(launch_kv8_reopen(kv->p8, inl, m, st));
          m = 0;
          break;
        }
    for (uint32_t l = 0; l < kv->d.n_layers; l++) {
      if (!take_back(kv, seqs[i], l, lens[i], &inl.r[m])) continue;
      if (++m < kKv8Inline) continue;
      KV_TRY(launch_kv8_reopen(kv->p8, inl, m, st));
      m = 0;
    }
  }
  if (m) KV_TRY(launch_kv8_reopen(kv->p8, inl, m, st));
  return GMOE_OK;
}

// Plans the call's entries and commits them (lengths advance and pages are taken only when
// the whole call fits), then queues the launches.
gmoe_status attend(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, const float* q, const float* k,
                   const float* v, float* out, hipStream_t st, uint32_t q_stride = 0, uint32_t kv_stride = 0) {
  if (kv->q8) return guarded([&] { return attend8(kv, layer, seqs, n, q, k, v, out, st, q_stride, kv_stride); });
  std::vector<AttnEntry> ent(n ? n : 1);
  uint32_t maxspan;
  bool distinct;
  if (gmoe_status s = plan(kv, layer, seqs, n, ent.data(), &maxspan, &distinct)) return s;
  const Runs R = find_runs(kv, ent.data(), n, out);
  const uint32_t ntile = (uint32_t)R.tiles.size(), npick = ntile ? (uint32_t)R.singles.size() : 0;
  uint32_t nchunk = (maxspan + kAttnChunk - 1) / kAttnChunk, skeys = 0;
  if (ntile) {
    skeys = split_key_tiles(kv, ntile, R.span) * kAttnTileKeys;
    nchunk = (R.span + skeys - 1) / skeys;
  }
  AttnLayout l = layout(kv, n, nchunk);
  const size_t o_rest = (l.total + 255) & ~(size_t)255;  // the singles' partials
  if (npick) l.total = o_rest + (size_t)npick * kv->d.n_heads * R.chunks * (kv->d.head_dim + 2) * 4;
  if (gmoe_status s = grow_scratch(kv, l.total)) return s;
  const size_t eb = n * sizeof(AttnEntry), tb = ntile * sizeof(AttnTile), pb = npick * sizeof(uint32_t);
  uint8_t* pin = nullptr;
  if (n > kAttnInline)
    if (gmoe_status s = take_pinned(kv, eb + tb + pb, st, &pin)) return s;
  commit(kv, layer, seqs, n, ent.data());
  for (uint32_t i = 0; i < npick; i++) ent[R.singles[i]].fresh |= kAttnSingle;
  AttnArgs a = args(kv, n, nchunk, l, q, k, v, out, q_stride, kv_stride);
  if (n <= kAttnInline) {  // a decode batch: the entries ride in the kernel arguments
    std::copy(ent.begin(), ent.begin() + n, a.inl);
    a.ent = nullptr;
  } else {
    memcpy(pin, ent.data(), eb);
    uint8_t* dev = kv->scratch + l.o_ent;
    a.ent = reinterpret_cast<const AttnEntry*>(dev);
    if (ntile) {
      memcpy(pin + eb, R.tiles.data(), tb);
      if (pb) memcpy(pin + eb + tb, R.singles.data(), pb);
      a.tiles = reinterpret_cast<const AttnTile*>(dev + eb);
      a.hent = reinterpret_cast<const AttnEntry*>(pin);
      a.htile = reinterpret_cast<const AttnTile*>(pin + eb);
      a.ntile = ntile;
      a.skeys = skeys;
      if (npick) {
        a.pick = reinterpret_cast<const uint32_t*>(dev + eb + tb);
        a.hpick = reinterpret_cast<const uint32_t*>(pin + eb + tb);
        a.npick = npick;
      }
      AttnArgs rest = a;
      rest.part = reinterpret_cast<float*>(kv->scratch + o_rest);
      rest.nchunk = R.chunks;
      KV_TRY(launch_attention_tiled(a, rest, st));
      return GMOE_OK;
    }
    KV_TRY(hipMemcpyAsync(dev, pin, eb, hipMemcpyHostToDevice, st));
  }
  a.distinct = distinct ? 1 : 0;
  KV_TRY(launch_attention(a, st));
  return GMOE_OK;
}

}  // namespace

namespace gmoe {

// For the decode-step driver (gmoe_model.cpp): the cache's widths, and whether each of
// the (distinct) sequences can take one more position in every layer, refused before
// any layer has run (as logits_batch refuses, llama/mod.rs:1163-1176).
void kv_dims(gmoe_kv* kv, uint32_t* n_layers, uint32_t* q_dim, uint32_t* kv_dim) {
  *n_layers = kv->d.n_layers;
  *q_dim = kv->d.n_heads * kv->d.head_dim;
  *kv_dim = kv->kvd;
}

// Attention over rows of q, k and v that sit q_stride and kv_stride floats apart (the
// model step's stacked q|k|v projection), queued on st.
gmoe_status kv_attend(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, const float* q, const float* k,
                      const float* v, uint32_t q_stride, uint32_t kv_stride, float* out, hipStream_t st) {
  std::lock_guard<std::mutex> g(kv->mu);
  KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
  return attend(kv, layer, seqs, n, q, k, v, out, st, q_stride, kv_stride);
}

gmoe_status kv_check_step(gmoe_kv* kv, const uint32_t* seqs, uint32_t n) {
  std::lock_guard<std::mutex> g(kv->mu);
  const gmoe_kv_desc& D = kv->d;
  uint64_t pages = 0;
  for (uint32_t i = 0; i < n; i++) {
    const uint32_t s = seqs[i];
    if (s >= kv->seqs.size() || !kv->seqs[s].open) return kfail(GMOE_ERR_INFERENCE, "sequence %u is not open", s);
    for (uint32_t j = 0; j < i; j++)
      if (seqs[j] == s) return kfail(GMOE_ERR_INFERENCE, "sequence %u appears twice in one decode step", s);
    for (uint32_t l = 0; l < D.n_layers; l++) {
      const uint32_t pos = kv->seqs[s].len[l];
      if (pos + 1 > D.max_positions)
        return kfail(GMOE_ERR_CACHE, "context window of %u positions is exhausted", D.max_positions);
      if (pos % D.block_size == 0) pages++;
    }
  }
  if (pages > kv->free_pages.size())
    return kfail(GMOE_ERR_CACHE, "the KV pool has %zu free pages, the step needs %llu", kv->free_pages.size(),
                 (unsigned long long)pages);
  return GMOE_OK;
}

// A prefill of n positions of one sequence (forward_tail, llama/mod.rs:1058-1066): the
// window and the pool checked for every layer before any layer runs.
gmoe_status kv_check_prefill(gmoe_kv* kv, uint32_t seq, uint32_t n) {
  std::lock_guard<std::mutex> g(kv->mu);
  const gmoe_kv_desc& D = kv->d;
  if (seq >= kv->seqs.size() || !kv->seqs[seq].open) return kfail(GMOE_ERR_INFERENCE, "sequence %u is not open", seq);
  uint64_t pages = 0;
  for (uint32_t l = 0; l < D.n_layers; l++) {
    const uint32_t len = kv->seqs[seq].len[l];
    if ((uint64_t)len + n > D.max_positions)
      return kfail(GMOE_ERR_CACHE, "%u tokens do not fit the %u-position context window (%u used)", n,
                   D.max_positions, len);
    for (uint64_t p = len; p < (uint64_t)len + n; p++)
      if (p % D.block_size == 0) pages++;
  }
  if (pages > kv->free_pages.size())
    return kfail(GMOE_ERR_CACHE, "the KV pool has %zu free pages, the prefill needs %llu", kv->free_pages.size(),
                 (unsigned long long)pages);
  return GMOE_OK;
}

// For decode steps replayed from a HIP graph (gmoe_model.cpp): the host plans every
// layer's entries (kv_plan_step), reserves the attention scratch, then commits them
// (kv_commit_step) and copies them to device memory the graph's attention launches read
// (kv_attend_dev). Those launches span a fixed number of chunks, the step's longest span
// rounded up to a power of two (kv_step_chunks), so one graph serves every step until a
// sequence outgrows the bucket; chunks past an entry's span are empty and merge as
// nothing, so the result is the same as over the entry's own chunks. kv_graph_chunks is
// the most a sequence can reach.
uint32_t kv_graph_chunks(gmoe_kv* kv) {
  const gmoe_kv_desc& D = kv->d;
  const uint32_t span = D.sliding_window ? std::min(D.sliding_window, D.max_positions) : D.max_positions;
  return (span + kAttnChunk - 1) / kAttnChunk;
}

uint32_t kv_step_chunks(gmoe_kv* kv, uint32_t maxspan) {
  const uint32_t need = (maxspan + kAttnChunk - 1) / kAttnChunk;
  uint32_t b = 1;
  while (b < need) b *= 2;
  return std::min(b, kv_graph_chunks(kv));
}

// Every layer's entries of a step (ents[l * stride + i]), planned but not committed, and
// the longest span any of them attends.
gmoe_status kv_plan_step(gmoe_kv* kv, const uint32_t* seqs, uint32_t n, AttnEntry* ents, size_t stride,
                         uint32_t* maxspan) {
  std::lock_guard<std::mutex> g(kv->mu);
  *maxspan = 1;
  for (uint32_t l = 0; l < kv->d.n_layers; l++) {
    uint32_t ms;
    if (gmoe_status s = plan(kv, l, seqs, n, ents + (size_t)l * stride, &ms)) return s;
    *maxspan = std::max(*maxspan, ms);
  }
  return GMOE_OK;
}

void kv_commit_step(gmoe_kv* kv, const uint32_t* seqs, uint32_t n, AttnEntry* ents, size_t stride) {
  std::lock_guard<std::mutex> g(kv->mu);
  for (uint32_t l = 0; l < kv->d.n_layers; l++) commit(kv, l, seqs, n, ents + (size_t)l * stride);
}

// A sequence's open rows, every layer's.
static size_t open_bytes(const gmoe_kv* kv) { return (size_t)kv->d.n_layers * 2 * kKv8Block * kv->kvd * 4; }

// The step's sequences as they stand (every layer's length and page count), and their
// return to it: pages taken since go back to the free list, lengths go back. A step that
// fails after committing positions restores them, so a refused step leaves every sequence
// where it was.
gmoe_status kv_snapshot(gmoe_kv* kv, const uint32_t* seqs, uint32_t n, std::vector<uint32_t>& snap, bool prompt) {
  std::lock_guard<std::mutex> g(kv->mu);
  snap.clear();
  // a prompt's rows move a sequence's open rows on to later blocks (a decode step's, at most
  // to one that it begins): copied before, so that a failed prompt can put them back
  if (kv->q8 && prompt) {
    const size_t bytes = open_bytes(kv);
    KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
    if (!kv->saved) KV_TRY(hipMalloc(&kv->saved, bytes));
    KV_TRY(hipMemcpyAsync(kv->saved, kv->p8.open + seqs[0] * (bytes / 4), bytes, hipMemcpyDeviceToDevice,
                          ctx_stream(kv->ctx)));
  }
  for (uint32_t i = 0; i < n; i++) {
    const Seq& S = kv->seqs[seqs[i]];
    for (uint32_t l = 0; l < kv->d.n_layers; l++) {
      snap.push_back(S.len[l]);
      snap.push_back((uint32_t)S.pages[l].size());
      snap.push_back(S.open_block[l]);
    }
  }
  return GMOE_OK;
}

void kv_restore(gmoe_kv* kv, const uint32_t* seqs, uint32_t n, const std::vector<uint32_t>& snap, bool prompt) {
  std::lock_guard<std::mutex> g(kv->mu);
  if (kv->q8 && prompt) {
    const size_t bytes = open_bytes(kv);
    (void)hipMemcpyAsync(kv->p8.open + seqs[0] * (bytes / 4), kv->saved, bytes, hipMemcpyDeviceToDevice,
                         ctx_stream(kv->ctx));
  }
  size_t at = 0;
  for (uint32_t i = 0; i < n && at + 3 * kv->d.n_layers <= snap.size(); i++) {
    Seq& S = kv->seqs[seqs[i]];
    for (uint32_t l = 0; l < kv->d.n_layers; l++, at += 3) {
      S.len[l] = snap[at];
      // a step leaves the open rows at its token's block: earlier ones come back from codes
      if (prompt) S.open_block[l] = snap[at + 2];
      while (S.pages[l].size() > snap[at + 1]) {
        kv->free_pages.push_back(S.pages[l].back());
        S.pages[l].pop_back();
      }
    }
  }
}


// Scratch of a decode step of n sequences over nchunk chunks.
static size_t step_bytes(const gmoe_kv* kv, uint32_t n, uint32_t nchunk) {
  return kv->q8 ? step8_bytes(kv, n, kv8_parts(nchunk * kAttnChunk)) : layout(kv, n, nchunk).total;
}

gmoe_status kv_reserve(gmoe_kv* kv, uint32_t n, uint32_t nchunk) {
  std::lock_guard<std::mutex> g(kv->mu);
  KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
  if (kv->fail_reserves) {
    kv->fail_reserves--;
    return kfail(GMOE_ERR_DEVICE, "attention scratch of %zu bytes: allocation refused (test hook)",
                 step_bytes(kv, n, nchunk));
  }
  if (kv->q8)
    if (gmoe_status s = grow_done(kv, n)) return s;
  return grow_scratch(kv, step_bytes(kv, n, nchunk));
}

const void* kv_scratch_id(gmoe_kv* kv) { return (const void*)kv->scratch_id; }

gmoe_status kv_plan_commit(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, AttnEntry* ent) {
  std::lock_guard<std::mutex> g(kv->mu);
  uint32_t maxspan;
  if (gmoe_status s = plan(kv, layer, seqs, n, ent, &maxspan)) return s;
  commit(kv, layer, seqs, n, ent);
  return GMOE_OK;
}

gmoe_status kv_attend_dev(gmoe_kv* kv, uint32_t n, const AttnEntry* d_ent, uint32_t nchunk, const float* q,
                          const float* k, const float* v, uint32_t q_stride, uint32_t kv_stride, float* out,
                          hipStream_t st, uint32_t nsl, uint64_t sl_stride) {
  std::lock_guard<std::mutex> g(kv->mu);
  if (kv->q8) {
    if (nsl > kMaxKsg) return kfail(GMOE_ERR_INFERENCE, "%u K slices exceed %u", nsl, kMaxKsg);
    Kv8Args a = args8(kv, n, q, k, v, out, q_stride, kv_stride);
    a.ent = d_ent;
    a.nsl = nsl;
    a.sl_stride = sl_stride;
    a.part = reinterpret_cast<float*>(kv->scratch);
    a.nparts = kv8_parts(nchunk * kAttnChunk);
    a.items = n * a.nparts;
    a.fused = kv8_fused(a.items, kv->d.n_kv_heads, a.nparts, kv->d.n_heads / kv->d.n_kv_heads * kv->d.head_dim);
    if (step_bytes(kv, n, nchunk) > kv->scratch_bytes || (size_t)n * kv->d.n_kv_heads > kv->n_done)
      return kfail(GMOE_ERR_INFERENCE, "attention scratch not reserved");
    KV_TRY(launch_kv8_step(a, Kv8Inline{}, st));
    return GMOE_OK;
  }
  const AttnLayout l = layout(kv, n, nchunk);
  if (l.total > kv->scratch_bytes) return kfail(GMOE_ERR_INFERENCE, "attention scratch not reserved");
  if (nsl > kMaxKsg) return kfail(GMOE_ERR_INFERENCE, "%u K slices exceed %u", nsl, kMaxKsg);
  AttnArgs a = args(kv, n, nchunk, l, q, k, v, out, q_stride, kv_stride);
  a.ent = d_ent;
  a.distinct = 1;  // a decode step's sequences, which kv_check_step refuses twice
  a.nsl = nsl;
  a.sl_stride = sl_stride;
  KV_TRY(launch_attention(a, st));
  return GMOE_OK;
}

}  // namespace gmoe

extern "C" {

static gmoe_status kv_create(gmoe_ctx* ctx, const gmoe_kv_desc* desc, bool q8, gmoe_kv** out) {
  if (!ctx || !desc || !out) return kfail(GMOE_ERR_INFERENCE, "null context, descriptor or output");
  *out = nullptr;
  const gmoe_kv_desc& D = *desc;
  if (D.n_layers == 0 || D.n_heads == 0 || D.n_kv_heads == 0 || D.head_dim == 0 || D.block_size == 0 ||
      D.max_positions == 0 || D.max_seqs == 0 || D.max_pages == 0)
    return kfail(GMOE_ERR_CONFIG, "KV cache dimensions must be positive");
  if (D.n_heads % D.n_kv_heads || D.n_heads / D.n_kv_heads > kAttnMaxGroup)
    return kfail(GMOE_ERR_MODEL, "n_heads %u must be a multiple of n_kv_heads %u, at most %u per kv head", D.n_heads,
                 D.n_kv_heads, kAttnMaxGroup);
  if (D.head_dim % 4 || D.head_dim > kAttnMaxHd)
    return kfail(GMOE_ERR_MODEL, "head_dim %u must be a multiple of 4 and at most %u", D.head_dim, kAttnMaxHd);
  if (!(D.rope_theta > 0.0f)) return kfail(GMOE_ERR_CONFIG, "rope_theta must be positive");
  if (q8 && D.block_size % kKv8Block)
    return kfail(GMOE_ERR_MODEL, "block_size %u must be a multiple of %u, the positions that share a scale", D.block_size,
                 kKv8Block);
  // pages have numbers of 32 bits, and 2^48 bytes are more than any card's
  const double kvd = (double)D.n_kv_heads * D.head_dim;
  if (D.max_pages > 0xffffffffull || (double)D.max_pages * D.block_size * kvd > 0x1p48 ||
      (double)D.max_seqs * D.n_layers * std::max((double)D.max_positions / D.block_size, kvd) > 0x1p48)
    return kfail(GMOE_ERR_CONFIG, "a KV cache of %llu pages and %u sequences is too large",
                 (unsigned long long)D.max_pages, D.max_seqs);
  std::unique_ptr<gmoe_kv> kv(new gmoe_kv);
  kv->ctx = ctx;
  kv->d = D;
  kv->kvd = D.n_kv_heads * D.head_dim;
  kv->ppseq = (D.max_positions + D.block_size - 1) / D.block_size;
  kv->page_floats = 2ull * D.block_size * kv->kvd;
  KV_TRY(hipSetDevice(ctx_device(ctx)));
  KV_TRY(hipMalloc(&kv->tables, (size_t)D.max_seqs * D.n_layers * kv->ppseq * 4));
  kv->q8 = q8;
  Kv8Pool& P = kv->p8;
  P.tables = kv->tables;
  P.n_kv = D.n_kv_heads;
  P.hd = D.head_dim;
  P.hdp = kv8_width(D.head_dim);
  P.bs = D.block_size;
  P.ppseq = kv->ppseq;
  if (q8) {
    const size_t units = D.max_pages * (D.block_size / kKv8Block) * D.n_kv_heads;
    KV_TRY(hipMalloc(&P.codes, units * 2 * kKv8Block * P.hdp));
    KV_TRY(hipMalloc(&P.scales, units * 2 * sizeof(float)));
    KV_TRY(hipMalloc(&P.open, (size_t)D.max_seqs * D.n_layers * 2 * kKv8Block * kv->kvd * 4));
    std::vector<double> turns(D.head_dim / 2);
    for (uint32_t i = 0; i < turns.size(); i++)
      turns[i] = std::pow((double)D.rope_theta, -(2.0 * i) / D.head_dim) / 6.283185307179586476925286766559;
    KV_TRY(hipMalloc((void**)&P.turns, turns.size() * sizeof(double)));
    KV_TRY(hipMemcpy(const_cast<double*>(P.turns), turns.data(), turns.size() * sizeof(double), hipMemcpyHostToDevice));
  } else {
    KV_TRY(hipMalloc(&kv->pool, D.max_pages * kv->page_floats * 4));
  }
  for (auto& e : kv->pin_ev) KV_TRY(hipEventCreateWithFlags(&e, hipEventDisableTiming));
  kv->free_pages.resize(D.max_pages);
  for (uint64_t i = 0; i < D.max_pages; i++) kv->free_pages[i] = (uint32_t)(D.max_pages - 1 - i);  // pops 0 first
  kv->seqs.resize(D.max_seqs);
  *out = kv.release();
  return GMOE_OK;
}

gmoe_status gmoe_kv_create(gmoe_ctx* ctx, const gmoe_kv_desc* desc, gmoe_kv** out) {
  return guarded([&] { return kv_create(ctx, desc, false, out); });
}

gmoe_status gmoe_kv_create_q8(gmoe_ctx* ctx, const gmoe_kv_desc* desc, gmoe_kv** out) {
  return guarded([&] { return kv_create(ctx, desc, true, out); });
}

void gmoe_kv_destroy(gmoe_kv* kv) {
  if (!kv) return;
  hipSetDevice(ctx_device(kv->ctx));
  hipDeviceSynchronize();  // queued calls may still use its buffers
  delete kv;
}

gmoe_status gmoe_kv_seq_open(gmoe_kv* kv, uint32_t* seq) {
  if (!kv || !seq) return kfail(GMOE_ERR_INFERENCE, "null cache or output");
  std::lock_guard<std::mutex> g(kv->mu);
  for (uint32_t s = 0; s < kv->seqs.size(); s++)
    if (!kv->seqs[s].open) {
      Seq& S = kv->seqs[s];
      S.open = true;
      S.len.assign(kv->d.n_layers, 0);
      S.pages.assign(kv->d.n_layers, {});
      S.open_block.assign(kv->d.n_layers, 0);
      *seq = s;
      return GMOE_OK;
    }
  return kfail(GMOE_ERR_CACHE, "all %u sequences are open", kv->d.max_seqs);
}

gmoe_status gmoe_kv_seq_close(gmoe_kv* kv, uint32_t seq) {
  if (!kv) return kfail(GMOE_ERR_INFERENCE, "null cache");
  std::lock_guard<std::mutex> g(kv->mu);
  if (seq >= kv->seqs.size() || !kv->seqs[seq].open) return kfail(GMOE_ERR_INFERENCE, "sequence %u is not open", seq);
  KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
  KV_TRY(hipDeviceSynchronize());  // queued calls may still read its pages
  Seq& S = kv->seqs[seq];
  for (auto& pl : S.pages)
    for (uint32_t p : pl) kv->free_pages.push_back(p);
  S = Seq{};
  return GMOE_OK;
}

gmoe_status gmoe_kv_seq_len(const gmoe_kv* kv, uint32_t seq, uint32_t layer, uint32_t* len) {
  if (!kv || !len) return kfail(GMOE_ERR_INFERENCE, "null cache or output");
  if (seq >= kv->seqs.size() || !kv->seqs[seq].open) return kfail(GMOE_ERR_INFERENCE, "sequence %u is not open", seq);
  if (layer >= kv->d.n_layers) return kfail(GMOE_ERR_INFERENCE, "layer %u of %u", layer, kv->d.n_layers);
  *len = kv->seqs[seq].len[layer];
  return GMOE_OK;
}

gmoe_status gmoe_kv_free_pages(gmoe_kv* kv, uint64_t* pages) {
  if (!kv || !pages) return kfail(GMOE_ERR_INFERENCE, "null cache or output");
  std::lock_guard<std::mutex> g(kv->mu);
  *pages = kv->free_pages.size();
  return GMOE_OK;
}

gmoe_status gmoe_kv_fail_reserves(gmoe_kv* kv, uint32_t count) {
  if (!kv) return kfail(GMOE_ERR_INFERENCE, "null cache");
  std::lock_guard<std::mutex> g(kv->mu);
  kv->fail_reserves = count;
  return GMOE_OK;
}

gmoe_status gmoe_attention(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, const float* q,
                           const float* k, const float* v, float* context) {
  if (!kv || !q || !k || !v || !context) return kfail(GMOE_ERR_INFERENCE, "null cache or activation pointer");
  std::lock_guard<std::mutex> g(kv->mu);
  KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
  const gmoe_kv_desc& D = kv->d;
  const size_t qb = (size_t)n * D.n_heads * D.head_dim * 4, kb = (size_t)n * kv->kvd * 4;
  float* buf = nullptr;
  KV_TRY(hipMalloc(&buf, 2 * qb + 2 * kb));
  float *dq = buf, *dk = buf + qb / 4, *dv = dk + kb / 4, *dout = dv + kb / 4;
  hipStream_t st = ctx_stream(kv->ctx);
  hipError_t e = hipMemcpyAsync(dq, q, qb, hipMemcpyHostToDevice, st);
  if (e == hipSuccess) e = hipMemcpyAsync(dk, k, kb, hipMemcpyHostToDevice, st);
  if (e == hipSuccess) e = hipMemcpyAsync(dv, v, kb, hipMemcpyHostToDevice, st);
  gmoe_status s = e == hipSuccess ? attend(kv, layer, seqs, n, dq, dk, dv, dout, st)
                                  : kfail(GMOE_ERR_DEVICE, "attention inputs: %s", hipGetErrorString(e));
  if (s == GMOE_OK) {
    e = hipMemcpyAsync(context, dout, qb, hipMemcpyDeviceToHost, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    if (e != hipSuccess) s = kfail(GMOE_ERR_DEVICE, "attention: %s", hipGetErrorString(e));
  }
  hipStreamSynchronize(st);
  hipFree(buf);
  return s;
}

gmoe_status gmoe_attention_async(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, const float* d_q,
                                 const float* d_k, const float* d_v, float* d_context, void* stream) {
  if (!kv || !d_q || !d_k || !d_v || !d_context) return kfail(GMOE_ERR_INFERENCE, "null cache or activation pointer");
  std::lock_guard<std::mutex> g(kv->mu);
  KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
  return attend(kv, layer, seqs, n, d_q, d_k, d_v, d_context, stream ? (hipStream_t)stream : ctx_stream(kv->ctx));
}

gmoe_status gmoe_kv_append(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, const float* k,
                           const float* v) {
  if (!kv || !k || !v) return kfail(GMOE_ERR_INFERENCE, "null cache, keys or values");
  if (n == 0) return kfail(GMOE_ERR_INFERENCE, "empty append");
  std::lock_guard<std::mutex> g(kv->mu);
  KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
  const size_t kb = (size_t)n * kv->kvd * 4;
  float* buf = nullptr;
  KV_TRY(hipMalloc(&buf, 2 * kb));
  hipStream_t st = ctx_stream(kv->ctx);
  hipError_t e = hipMemcpyAsync(buf, k, kb, hipMemcpyHostToDevice, st);
  if (e == hipSuccess) e = hipMemcpyAsync(buf + kb / 4, v, kb, hipMemcpyHostToDevice, st);
  gmoe_status s = e == hipSuccess ? guarded([&] { return append(kv, layer, seqs, n, buf, buf + kb / 4, st); })
                                  : kfail(GMOE_ERR_DEVICE, "append inputs: %s", hipGetErrorString(e));
  e = hipStreamSynchronize(st);
  hipFree(buf);
  if (s == GMOE_OK && e != hipSuccess) s = kfail(GMOE_ERR_DEVICE, "append: %s", hipGetErrorString(e));
  return s;
}

gmoe_status gmoe_kv_append_async(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, uint32_t n, const float* d_k,
                                 const float* d_v, void* stream) {
  if (!kv || !d_k || !d_v) return kfail(GMOE_ERR_INFERENCE, "null cache, keys or values");
  if (n == 0) return kfail(GMOE_ERR_INFERENCE, "empty append");
  std::lock_guard<std::mutex> g(kv->mu);
  KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
  const hipStream_t st = stream ? (hipStream_t)stream : ctx_stream(kv->ctx);
  return guarded([&] { return append(kv, layer, seqs, n, d_k, d_v, st); });
}

gmoe_status gmoe_kv_read(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, const uint32_t* pos, uint32_t n, float* k,
                         float* v) {
  if (!kv || !k || !v) return kfail(GMOE_ERR_INFERENCE, "null cache or outputs");
  if (n == 0) return kfail(GMOE_ERR_INFERENCE, "empty read");
  std::lock_guard<std::mutex> g(kv->mu);
  KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
  const size_t kb = (size_t)n * kv->kvd * 4;
  float* buf = nullptr;
  KV_TRY(hipMalloc(&buf, 2 * kb));
  hipStream_t st = ctx_stream(kv->ctx);
  gmoe_status s = guarded([&] { return read_rows(kv, layer, seqs, pos, n, buf, buf + kb / 4, st); });
  if (s == GMOE_OK) {
    hipError_t e = hipMemcpyAsync(k, buf, kb, hipMemcpyDeviceToHost, st);
    if (e == hipSuccess) e = hipMemcpyAsync(v, buf + kb / 4, kb, hipMemcpyDeviceToHost, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    if (e != hipSuccess) s = kfail(GMOE_ERR_DEVICE, "read: %s", hipGetErrorString(e));
  }
  hipStreamSynchronize(st);
  hipFree(buf);
  return s;
}

gmoe_status gmoe_kv_read_async(gmoe_kv* kv, uint32_t layer, const uint32_t* seqs, const uint32_t* pos, uint32_t n,
                               float* d_k, float* d_v, void* stream) {
  if (!kv || !d_k || !d_v) return kfail(GMOE_ERR_INFERENCE, "null cache or outputs");
  std::lock_guard<std::mutex> g(kv->mu);
  KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
  const hipStream_t st = stream ? (hipStream_t)stream : ctx_stream(kv->ctx);
  return guarded([&] { return read_rows(kv, layer, seqs, pos, n, d_k, d_v, st); });
}

gmoe_status gmoe_kv_truncate(gmoe_kv* kv, const uint32_t* seqs, const uint32_t* lens, uint32_t n, void* stream) {
  if (!kv) return kfail(GMOE_ERR_INFERENCE, "null cache");
  std::lock_guard<std::mutex> g(kv->mu);
  KV_TRY(hipSetDevice(ctx_device(kv->ctx)));
  const hipStream_t st = stream ? (hipStream_t)stream : ctx_stream(kv->ctx);
  return guarded([&] { return truncate(kv, seqs, lens, n, st); });
}

}  // extern "C"
