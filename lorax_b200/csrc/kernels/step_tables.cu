// Tables of a ragged step from its sequences' lengths: per-token positions, cache slots and adapter slots, padded block tables, the lists of
// attention tiles and of adapter tiles.
//
//   seqs    [4, B]: tokens n, cached tokens c, adapter slot a (-1: none), pages p of every sequence; pages: the page lists end to end
//   cu[b]   = sum of n over the sequences before b;  off[b] = the same of p
//   table[b, j] = pages[off + j] for j < p; pages[off + j mod p] where a sliding window recycles them; else 0
//   token t of sequence b (the last whose cu[b] <= t): position c + t - cu[b], slot table[b, position / page] * page + position mod page
//   tiles of height h: (b, 0), (b, h), (b, 2 h) ... below n, for every sequence in turn
//   adapter tiles: (a, row_offset + cu[b] + first row, rows, 0) of at most `lora_rows` rows, for the sequences that have an adapter
//
// The reference assembles these arrays on the host for every batch (server/lorax_server/models/flash_causal_lm.py:200-420).
//
// Bound by latency: a few KB to a few MB.  One launch, in which every block sums up the sequences' lengths by itself (B <= 4096: 16 KB that
// stay in L2) instead of waiting for another one's sums, and writes 1024 entries of one of the outputs.
#include "common.cuh"

namespace lx {

constexpr int kTablesThreads = 256;
constexpr int kTablesPer = 1024;          // entries of an output that a block writes
constexpr int kTablesMaxSeqs = 4096;
constexpr int kTablesLists = 4;
constexpr int kTablesMaxTiles = 1 << 30;  // entries of a list (its blocks count in 32 bits, past its end)

struct TileList {
  int* seq;
  int* q0;
  int height, count;
};

struct StepTablesParams {
  const int* seqs;         // [4, B], rows `ld` apart
  long long ld;
  const int* pages;
  int num_pages, B, T, M, page, window, row_offset;
  int* cu_q;
  int* positions;
  int* slots;
  int* tok_slot;
  int* tables;
  TileList lists[kTablesLists];
  int nlists;
  const int4* lead;        // tiles that precede the step's own, or null
  int nlead, lora_rows, lora_count;
  int4* lora;              // [nlead + lora_count]
  int first[3 + kTablesLists];      // first block of: tables, lists .., adapter tiles; blocks in front of first[0] write tokens
};

// sums[b] = sum of f(i) over i < b, for b = 0 .. B.
template <typename F>
LX_DEVICE void tables_scan(int* sums, int* warps, int B, F&& f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int carry = 0;
  for (int b0 = 0; b0 < B; b0 += kTablesThreads) {
    const int b = b0 + threadIdx.x, own = b < B ? f(b) : 0;
    int v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warps[warp] = v;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < kTablesThreads / 32; ++i) {
      if (i < warp) v += warps[i];
      total += warps[i];
    }
    if (b < B) sums[b] = carry + v - own;
    carry += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) sums[B] = carry;
  __syncthreads();
}

// The last b < B with sums[b] <= i.
LX_DEVICE int tables_find(const int* sums, int B, int i) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

// Lengths, places and page counts below zero count as zero.
LX_DEVICE int tables_len(const StepTablesParams& p, int row, int b) { return max(p.seqs[row * p.ld + b], 0); }

// Tiles of `height` that n tokens make.
LX_DEVICE int tables_up(int n, int height) { return n / height + (n % height != 0); }

LX_DEVICE int tables_entry(const StepTablesParams& p, int off, int held, int j) {
  if (j < 0) return 0;                    // (a place past 32 bits)
  if (j >= held) {
    const bool recycled = p.window > 0 && held > 0 && held < p.M && (long long)held * p.page >= (long long)p.window + p.page;
    if (!recycled) return 0;
    j %= held;
  }
  const unsigned at = (unsigned)off + (unsigned)j;      // (of page counts whose sum is past 32 bits nothing is read out of range)
  return at < (unsigned)p.num_pages ? p.pages[at] : 0;
}

__global__ void __launch_bounds__(kTablesThreads) step_tables_kernel(const __grid_constant__ StepTablesParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ int sums[];           // two rows of B + 1
  __shared__ int warps[kTablesThreads / 32];
  const int block = blockIdx.x;
  int* const cu = sums;
  int* const off = sums + p.B + 1;
  auto tokens = [&](int b) { return tables_len(p, 0, b); };
  auto held = [&](int b) { return tables_len(p, 3, b); };
  if (block < p.first[0]) {               // tokens
    tables_scan(cu, warps, p.B, tokens);
    tables_scan(off, warps, p.B, held);
    if (block == 0)
      for (int b = threadIdx.x; b <= p.B; b += kTablesThreads) p.cu_q[b] = cu[b];
#pragma unroll
    for (int i = 0; i < kTablesPer / kTablesThreads; ++i) {
      const int t = block * kTablesPer + i * kTablesThreads + threadIdx.x;
      if (t >= p.T) break;
      int pos = 0, slot = -1, adapter = -1;
      if (t < cu[p.B]) {
        const int b = tables_find(cu, p.B, t);
        pos = tables_len(p, 1, b) + t - cu[b];
        slot = tables_entry(p, off[b], held(b), min(pos / p.page, p.M - 1)) * p.page + pos % p.page;
        adapter = p.seqs[2 * p.ld + b];
      }
      p.positions[t] = pos;
      p.slots[t] = slot;
      p.tok_slot[t] = adapter;
    }
    return;
  }
  if (block < p.first[1]) {               // block tables
    tables_scan(off, warps, p.B, held);
    const long long at = (long long)(block - p.first[0]) * kTablesPer, all = (long long)p.B * p.M;
#pragma unroll
    for (int i = 0; i < kTablesPer / kTablesThreads; ++i) {
      const long long e = at + i * kTablesThreads + threadIdx.x;
      if (e >= all) break;
      const int b = (int)(e / p.M), j = (int)(e - (long long)b * p.M);
      p.tables[e] = tables_entry(p, off[b], held(b), j);
    }
    return;
  }
  for (int l = 0; l < p.nlists; ++l) {
    if (block >= p.first[2 + l]) continue;
    const TileList list = p.lists[l];
    tables_scan(cu, warps, p.B, [&](int b) { return tables_up(tokens(b), list.height); });
    for (int i = (block - p.first[1 + l]) * kTablesPer + threadIdx.x, end = min(list.count, i - (int)threadIdx.x + kTablesPer); i < end; i += kTablesThreads) {
      const bool live = i < cu[p.B];
      const int b = live ? tables_find(cu, p.B, i) : -1;
      list.seq[i] = b;
      list.q0[i] = live ? (i - cu[b]) * list.height : 0;
    }
    return;
  }
  tables_scan(cu, warps, p.B, tokens);    // adapter tiles
  int* const tiles = off;
  tables_scan(tiles, warps, p.B, [&](int b) { return p.seqs[2 * p.ld + b] < 0 ? 0 : tables_up(tokens(b), p.lora_rows); });
  const int n = p.nlead + p.lora_count;
  for (int i = (block - p.first[1 + p.nlists]) * kTablesPer + threadIdx.x, end = min(n, i - (int)threadIdx.x + kTablesPer); i < end; i += kTablesThreads) {
    int4 tile = make_int4(-1, 0, 0, 0);
    if (i < p.nlead) {
      tile = p.lead[i];
    } else if (i - p.nlead < tiles[p.B]) {
      const int b = tables_find(tiles, p.B, i - p.nlead), row = (i - p.nlead - tiles[b]) * p.lora_rows;
      tile = make_int4(p.seqs[2 * p.ld + b], p.row_offset + cu[b] + row, min(p.lora_rows, tokens(b) - row), 0);
    }
    p.lora[i] = tile;
  }
}

}  // namespace lx

extern "C" {

int lx_step_tables_max_seqs() { return lx::kTablesMaxSeqs; }

// `out` (16-byte aligned) takes the outputs end to end: adapter tiles [nlead + lora_count, 4], cu_q [B + 1], positions, slots, tok_slot [T] each,
// tables [B, M], then seq and q0 [counts[l]] of every list.  The counts are the caller's; entries past what the lengths make hold: positions 0,
// slots and adapter slots -1, tiles of sequence or adapter -1.  What the lengths make beyond them is left out.
int lx_step_tables(const int* seqs, long long ld, const int* pages, int num_pages, int B, int T, int M, int page, int window, int row_offset,
                   const int* heights, const int* counts, int nlists, const int* lead, int nlead, int lora_rows, int lora_count, int* out,
                   void* stream) {
  using namespace lx;
  if (B < 0 || B > kTablesMaxSeqs || T < 0 || M <= 0 || page <= 0 || num_pages < 0 || nlists < 0 || nlists > kTablesLists || row_offset < 0 || nlead < 0 || lora_count < 0 || nlead > kTablesMaxTiles || lora_count > kTablesMaxTiles - nlead ||
      (lora_count > 0 && lora_rows <= 0) || (nlead > 0 && lead == nullptr))
    return -1;
  if ((reinterpret_cast<uintptr_t>(out) & 15) != 0 || (reinterpret_cast<uintptr_t>(lead) & 15) != 0) return -2;
  StepTablesParams p{};
  p.seqs = seqs; p.ld = ld; p.pages = pages; p.num_pages = num_pages;
  p.B = B; p.T = T; p.M = M; p.page = page; p.window = window; p.row_offset = row_offset;
  p.lead = reinterpret_cast<const int4*>(lead); p.nlead = nlead; p.lora_rows = lora_rows; p.lora_count = lora_count;
  p.lora = reinterpret_cast<int4*>(out);
  out += 4LL * (nlead + lora_count);
  p.cu_q = out; out += B + 1;
  p.positions = out; out += T;
  p.slots = out; out += T;
  p.tok_slot = out; out += T;
  p.tables = out; out += (long long)B * M;
  auto blocks = [](long long n) { return (n + kTablesPer - 1) / kTablesPer; };
  long long grid = T > 0 ? blocks(T) : 1;                      // (the first block writes cu_q)
  p.first[0] = (int)grid;
  grid += blocks((long long)B * M);
  p.first[1] = (int)grid;
  p.nlists = nlists;
  for (int l = 0; l < nlists; ++l) {
    if (heights[l] <= 0 || counts[l] < 0 || counts[l] > kTablesMaxTiles) return -1;
    p.lists[l] = TileList{out, out + counts[l], heights[l], counts[l]};
    out += 2LL * counts[l];
    grid += blocks(counts[l]);
    p.first[2 + l] = (int)grid;
  }
  grid += blocks(nlead + lora_count);
  if (grid > 0x7fffffffLL) return -1;
  launch_pdl(step_tables_kernel, dim3((unsigned)grid), dim3(kTablesThreads), 2 * (B + 1) * sizeof(int), reinterpret_cast<cudaStream_t>(stream), p);
  return -(int)cudaGetLastError();
}

}  // extern "C"
