// The maps of a step, made on the device from the requests' lengths and the pages they hold: where each row of
// the step goes (position, request, place in the cache), the padded block tables, the blocks of SCALE_TOKENS
// positions that the step writes (what the append to an 8-bit cache walks over) and the tiles of packed rows of the
// requests that bring more than a few (what its prompt attention walks over).
// The reference builds positions and row slots on the host, row by row, and copies them
// (cuongvng/bare-cuda-4gib engine/src/model.cpp:480-496; its page table is the host's too, engine/src/kv_cache.cpp:94-118).
//
//   q_start = exclusive sum of q_len          kv_len = cached + q_len
//   position = cached + place in the request  slot = page * page_tokens + position % page_tokens
//   table[s][b] = pages[first page of s + b]  for the ceil(kv_len / page_tokens) blocks of s, -1 behind them
//
// A request with cached < 0 is an idle row that pads a decode step: its rows count, it holds nothing.  Positions behind the table's
// last page are not held, and rows behind the step's last belong to no request: what is listed here is in bounds, whatever the lengths say.
//
// Nothing here is worth bandwidth (3 MB at most); what it costs is its chain of dependent trips to memory: lengths, then pages, then
// the stores.  So every block sums the lengths of all requests for itself (no block waits for another, no second launch), and
// the rows, table rows, blocks and tiles are dealt out over the grid.
// It is an ordinary launch, not a dependent one: it waits for all kernels before it, and no kernel behind it
// starts before it has ended, so kernels that read metadata ahead of their wait may read what it wrote.
// One B200: 8 decoding requests 4.0 us in a graph (6.3 a call after another from Python), 256 requests of up to 30,000 positions beside four
// prompts (3 MB of tables) 6.1 (8.2).

#include "cache8.cuh"

// What a call is made of (all arrays on the device; what they hold, see llm_step_maps).
struct MapsArgs {
  const int32_t* cached;
  const int32_t* q_len;
  int n_seqs;
  const int32_t* pages;
  int n_pages;
  int n_rows, page_tokens, group, tile_rows, few_rows, max_blocks, n_writes, n_tiles;
  int32_t *seq_q_start, *seq_q_len, *seq_kv_len, *order, *positions, *row_seq;
  long long* slots;
  int32_t *block_table, *write_seq, *write_block, *tile_seq, *tile_index;
};

namespace {

constexpr int THREADS = 256;
constexpr int TABLE_CHUNK = 256;     // entries of a table row that a warp fills at a time
constexpr int MAX_SEQS = 4096;       // the four sums of every request lie in shared memory

// What request s brings: rows, pages, written blocks, tiles.
__device__ __forceinline__ int4 counts_of(const MapsArgs& a, int s, int& cached, int& q) {
  cached = a.cached[s];
  q = min(max(a.q_len[s], 0), a.n_rows);
  const int blocks = cached < 0 ? 0 : (int)(((long long)cached + q + a.page_tokens - 1) / a.page_tokens);
  if (cached < 0 || q == 0) return make_int4(q, blocks, 0, 0);
  const int kv = cached + q, packed = q * a.group;
  return make_int4(q, blocks, (kv - 1) / SCALE_TOKENS - cached / SCALE_TOKENS + 1,
                   packed > a.few_rows ? (packed + a.tile_rows - 1) / a.tile_rows : 0);
}
__device__ __forceinline__ int4 add(int4 x, int4 y) { return make_int4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w); }
__device__ __forceinline__ int4 shift_up(int4 x, int by) {
  return make_int4(__shfl_up_sync(0xffffffffu, x.x, by), __shfl_up_sync(0xffffffffu, x.y, by), __shfl_up_sync(0xffffffffu, x.z, by),
                   __shfl_up_sync(0xffffffffu, x.w, by));
}

// The request whose stretch of `starts` (n + 1 ascending numbers) holds entry i; n if i lies behind the last.
__device__ __forceinline__ int whose(const int* starts, int n, int i) {
  int lo = 0, hi = n;                // the answer is the last s with starts[s] <= i and starts[s + 1] > i
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid + 1] <= i) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(THREADS) step_maps_kernel(const MapsArgs a) {
  extern __shared__ int sums[];      // [5][n_seqs + 1]: exclusive sums of rows, pages, written blocks, tiles; lengths after the step
  __shared__ int4 warp_total[THREADS / 32];
  const int S = a.n_seqs, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int *rows = sums, *first_page = rows + S + 1, *writes = first_page + S + 1, *tiles = writes + S + 1, *kv_len = tiles + S + 1;
  // each thread sums a stretch of requests, the block sums the stretches
  const int per = (S + THREADS - 1) / THREADS, s0 = min(S, tid * per), s1 = min(S, s0 + per);
  int4 mine = make_int4(0, 0, 0, 0);
  int cached, q;
  for (int s = s0; s < s1; ++s) mine = add(mine, counts_of(a, s, cached, q));
  int4 up = mine;
#pragma unroll
  for (int by = 1; by < 32; by <<= 1) {
    const int4 below = shift_up(up, by);
    if (lane >= by) up = add(up, below);
  }
  if (lane == 31) warp_total[warp] = up;
  __syncthreads();
  int4 at = make_int4(up.x - mine.x, up.y - mine.y, up.z - mine.z, up.w - mine.w);
  for (int w = 0; w < warp; ++w) at = add(at, warp_total[w]);
  for (int s = s0; s < s1; ++s) {
    rows[s] = at.x, first_page[s] = at.y, writes[s] = at.z, tiles[s] = at.w;
    const int4 c = counts_of(a, s, cached, q);
    q = cached < 0 ? 0 : min(q, max(a.n_rows - at.x, 0));
    kv_len[s] = cached < 0 ? 0 : cached + q;
    if (blockIdx.x == 0) {
      a.seq_q_start[s] = at.x;
      a.seq_q_len[s] = q;
      a.seq_kv_len[s] = cached < 0 ? 0 : cached + q;
    }
    at = add(at, c);
  }
  if (tid == THREADS - 1) rows[S] = at.x, first_page[S] = at.y, writes[S] = at.z, tiles[S] = at.w;
  __syncthreads();

  const int step = gridDim.x * THREADS, first = blockIdx.x * THREADS + tid;
  for (int i = first; i < a.n_rows; i += step) {
    const int s = whose(rows, S, i);
    int position = 0;
    long long slot = -1;
    if (s < S && a.cached[s] >= 0) {
      position = a.cached[s] + i - rows[s];
      const int b = position / a.page_tokens, at_page = first_page[s] + b;
      const int page = b < a.max_blocks && (unsigned)at_page < (unsigned)a.n_pages ? a.pages[at_page] : -1;
      if (page >= 0) slot = (long long)page * a.page_tokens + position % a.page_tokens;
    }
    a.positions[i] = position;
    a.row_seq[i] = s < S ? s : -1;
    a.slots[i] = slot;
  }
  for (int i = first; i < a.n_writes; i += step) {
    const int s = whose(writes, S, i);
    a.write_seq[i] = s < S ? s : -1;
    a.write_block[i] = s < S ? a.cached[s] / SCALE_TOKENS + i - writes[s] : 0;
  }
  for (int i = first; i < a.n_tiles; i += step) {
    const int s = whose(tiles, S, i);
    a.tile_seq[i] = s < S ? s : -1;
    a.tile_index[i] = s < S ? i - tiles[s] : 0;
  }
  // a request's place by length: how many are longer, or as long and come before it (a warp counts for one request)
  for (int s = first >> 5; s < S; s += step >> 5) {
    const int mine_len = kv_len[s];
    int before = 0;
    for (int o = lane; o < S; o += 32) before += kv_len[o] > mine_len || (kv_len[o] == mine_len && o < s);
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) a.order[before] = s;
  }
  // the tables: a warp takes a stretch of TABLE_CHUNK entries of a row at a time, all of its loads on their way at once
  const int chunks = (a.max_blocks + TABLE_CHUNK - 1) / TABLE_CHUNK;
  for (int c = first >> 5; c < S * chunks; c += step >> 5) {
    const int s = c / chunks, b0 = (c - s * chunks) * TABLE_CHUNK + lane, from = first_page[s], held = from < 0 ? 0 : min(first_page[s + 1], a.n_pages) - from;
    int32_t* row = a.block_table + (long long)s * a.max_blocks;
    int page[TABLE_CHUNK / 32];
#pragma unroll
    for (int i = 0; i < TABLE_CHUNK / 32; ++i) page[i] = b0 + 32 * i < held ? a.pages[from + b0 + 32 * i] : -1;
#pragma unroll
    for (int i = 0; i < TABLE_CHUNK / 32; ++i)
      if (b0 + 32 * i < a.max_blocks) row[b0 + 32 * i] = page[i];
  }
  __threadfence();      // what this thread wrote is there for all before its block has ended, and with it any kernel behind it can start
}

}  // namespace

extern "C" int llm_step_maps_max_seqs() { return MAX_SEQS; }

// Every output is a dense device array: per request (seq_q_start, seq_q_len, seq_kv_len, order), per row of the step (positions, row_seq,
// slots), [n_seqs][max_blocks] (block_table), and lists of n_writes and n_tiles entries, whose entries behind the last
// are -1 and 0.  `pages`: the held pages of request 0, then of request 1, ..., ceil(kv_len / page_tokens) each (-1: given back).
extern "C" int llm_step_maps(const MapsArgs* args, cudaStream_t stream) {
  const MapsArgs& a = *args;
  if (a.n_seqs <= 0) return 0;
  if (a.n_seqs > MAX_SEQS || a.page_tokens <= 0 || a.page_tokens % SCALE_TOKENS || a.group <= 0 || a.tile_rows <= 0 || a.max_blocks <= 0 ||
      a.few_rows < 0 || a.n_rows < 0 || a.n_writes < 0 || a.n_tiles < 0 || a.n_pages < 0)
    return ERR_BAD_SIZE;
  const size_t smem = (size_t)5 * (a.n_seqs + 1) * 4;
  static unsigned long long raised = 0;
  const unsigned long long here = device_bit();
  if (!(raised & here)) {
    if (cudaFuncSetAttribute(step_maps_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 5 * (MAX_SEQS + 1) * 4) != cudaSuccess)
      return launch_status();
    raised |= here;
  }
  // four numbers a thread, one block an SM at most
  const long long numbers = (long long)a.n_rows + a.n_writes + a.n_tiles + (long long)a.n_seqs * a.max_blocks;
  const long long blocks = (numbers + 4 * THREADS - 1) / (4 * THREADS);
  step_maps_kernel<<<(int)(blocks < 1 ? 1 : blocks > 148 ? 148 : blocks), THREADS, smem, stream>>>(a);
  return launch_status();
}
