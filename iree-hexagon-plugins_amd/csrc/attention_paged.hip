// Attention over a paged KV cache for a batch whose requests share a prefix.
//
// The new tokens of all requests are packed rows (row_starts); the query rows
// of a KV head are its `group` heads of every token, r = token * group + head.
// A row's keys are the prefix, which every row sees whole, and its request's
// own keys up to itself. Each is a run of pages named by a table. With
//   m = max_j s_j, l = sum_j 2^(s_j - m), a = sum_j 2^(s_j - m) v_j
// of any set of keys (s = q . k * scale * log2 e), two sets join as
//   m = max(m1, m2), l = l1 2^(m1 - m) + l2 2^(m2 - m), a alike, o = a / l,
// so the prefix can be computed for tiles of rows of the whole batch, each
// request's own keys for tiles of its own rows, and any tile's keys in pieces;
// a second kernel joins the parts of each row. Where requests bring enough
// rows to fill tiles, a tile walks the prefix and its own keys in turn.
//
// The tiles of a KV head, one after the other with the keys of each, are a
// line that a fixed number of workgroups share out evenly, whatever the
// lengths are: every workgroup finds its stretch of the line by itself. A tile
// that one workgroup has whole needs no joining.
//
// Tiles of up to 16 rows (a token or a few of a request): the 4 waves take
// blocks of 32 keys in turn, each alone: K rows go from memory into MFMA
// fragments (S^T = K Q^T; a lane holds 4 + 4 keys of one row), V rows through
// the wave's LDS tile, from which transposed reads take the key order that S^T
// has, so P stays in registers for O^T += V^T P. The next block's rows are in
// flight during the current one, and the page numbers of the one after it.
// They are bound by reading K and V: 64 requests' tokens behind 8192 keys (166
// MB) take 43 us and 5 us to join, 32 requests' without a prefix (209 MB) 44
// and 5, 4.7 TB/s.
// Wide tiles (128 rows, 32 a wave): K and V of 64 keys are copied straight
// into a two-slot LDS ring that all waves read, one barrier a block; two such
// workgroups share a CU, so one's softmax runs beside the other's MFMAs. They
// are bound by issuing: of a step's 4100 cycles the matrix cores are busy for
// 45 % (four prompts, 2243 rows of 32 heads behind 4096 keys: 193 GFLOP in 234
// to 244 us by card, 790 to 820 TFLOP/s, of which 17 us to join). Two barriers a
// step with copies further ahead took 263 us for the 239 of then, copies between
// the MFMAs 247.
// A call costs 7 us at least (launch 2, finding its place 2, a tile 3), and 4
// more where parts are joined.
//
// Trees (kTree): of its request's new tokens a row sees those before it whose bit
// its mask has. Only blocks that hold new tokens look: 64 bits of the mask, cut
// from words at any bit, go into the test that hides keys past a row's own
// (narrow tiles read them with the block's rows, ahead; wide ones where they use
// them, so that such a step also waits for the next block's copies). All blocks of
// a prompt without cached tokens are such ones: a chain of 1000, 32 / 8 heads of
// 128, takes 40.6 us, without masks 35.1; of 4096 217 and 184; of 1000 behind 4000
// cached tokens 110 and 102.
//
// Packed rows (kRows): keys are rows too, so a block's place is a base and its
// rows follow one another; there are no tables and no prefix. Where there are
// enough tiles none is split, and a kernel of its own gives each a workgroup, the
// longest first. A prompt of 8191 tokens, 32 heads over 8 of 128 (550 GFLOP),
// takes 540 to 570 us by card, 960 to 1020 TFLOP/s: the matrix cores are busy for
// 54 % of the cycles, at the 1.75 GHz that the clock falls to under them.
// Prompts of 7195 rows in 6 (79 GFLOP) take 109 to 118 us: of a tile's 30 us some
// 9 are its place, its first rows and its stores. Tried without gain or with too
// little: tiles of 256 rows with 64 rows a wave, softmax woven between the
// matrix instructions (560 -> 623 us); 8 waves of 32 rows in alternating phases
// on shared keys (3 % less from 3000 keys on, more below); K read 6 instructions
// ahead, no wave priorities, priority for a tile's start, 4 workgroups a CU of 64
// dims or a third slot of their ring (none better; most within 1 %).
#include <cstdio>

#include "attention_common.h"
#include "device_common.h"
#include "kernels_internal.h"

namespace ihp {

namespace {

constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = kPagedThreads / 64;
constexpr int kBlockKeys = 32;   // of a narrow tile's wave
constexpr int kStepKeys = 64;    // of a wide tile's block; pieces of a line
constexpr int kNarrowRows = 16;
constexpr int kWideRows = 128;
// How far (in log2) a wide tile's row maximum may pass its reference before
// the reference moves and O is rescaled: the sums are exact in either case,
// and the weights' roundings relative, so a lag of 4 is 0-5 % further from 64
// bits than none (rounding N(0, 1) scores and values of 64 to 5000 keys).
// (Four prompts of 2243 rows: 259.8 us with none, 241.3 with 4.)
constexpr float kLag = 4.0f;
constexpr int kTurnWgs = 256;  // workgroups that give every CU one
constexpr uint32_t kLevelKeys = 128;  // by which whole tiles are ordered
constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The same value in every lane, in scalar registers.
__device__ __forceinline__ int uniform(int x) {
  return __builtin_amdgcn_readfirstlane(x);
}

// A value kept in a scalar register: the compiler would read an argument again
// at its uses in a loop, and wait for it among the LDS reads.
template <typename T>
__device__ __forceinline__ T held(T x) {
  asm volatile("" : "+s"(x));
  return x;
}

// The kernel's arguments, read where they are used: held in registers from the
// kernel's start they pushed the tiles' own out of theirs.
__device__ __forceinline__ const PagedAttention &arguments() {
  auto *at = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *(const PagedAttention *)at;
}

// row_starts[b], within the rows that there are whatever it holds.
__device__ __forceinline__ int row_start(const PagedAttention &p, int b) {
  const int r = p.row_starts[b];
  return r < 0 ? 0 : r > p.rows ? p.rows : r;
}

// The token of a packed row: r / group, of rows below 2^30.
__device__ __forceinline__ int token_of(const PagedAttention &p, int r) {
  return p.group == 1 ? r
                      : (int)(__umulhi((uint32_t)r, p.group_magic) >>
                              p.group_shift);
}

// What the workgroup knows of the requests, in LDS: of lane l's `each`
// requests the first one's row starts and length, and the rows of small
// requests before them.
struct Requests {
  int of[4][64];  // kRows: the row of the first key last
  uint32_t small[64];
};

// Requests of up to so many rows share tiles of the prefix (one of more has tiles
// of its own and walks the prefix in them): those of a narrow tile, and trees
// that would leave much of a wide tile empty (24 trees of 3 to 114 rows a KV head
// behind 2048 keys: 51.2 -> 45.4 us, 46.7 with 64).
constexpr int kSmallRows = kNarrowRows;
template <PagedKeys KIND>
constexpr int kSharedRows = KIND == PagedKeys::kTree ? 96 : kSmallRows;

// One tile's work: rows r0 .. r_end - 1 (of a KV head; `compact`: the small
// requests' rows alone) against steps s_begin .. s_end - 1 of 64 keys, the
// first `lead` of them the prefix's.
struct PagedTile {
  int64_t key0;  // kRows: the row of the request's first key
  int kv_head, r0, r_end;
  bool compact;
  int lead;
  const int32_t *table;  // the request's pages
  int own_end;           // own keys that its pages hold
  int seen;              // own keys that the tile's last row sees
  int base, first;       // row r sees own keys .. base + r / group - first
  int s_begin, s_end;
  int64_t part;          // where row 0's part would be; -1: the result
};

// Own keys that row r sees.
__device__ __forceinline__ int sees(const PagedAttention &p,
                                    const PagedTile &t, int r) {
  const int64_t n = (int64_t)t.base + token_of(p, r) - t.first + 1;
  return n < 0 ? 0 : n > t.own_end ? t.own_end : (int)n;
}

// What a row's mask says of the KEYS own keys from key0, bit i of key key0 + i.
// New token j of the request is key t.base + j: those below 0 are cached, those
// from 32 * words on have no bit, and neither are hidden here.
struct TreeWords {
  uint32_t w[3];
};
template <int KEYS>
__device__ __forceinline__ TreeWords tree_words(const PagedAttention &p,
                                                const PagedTile &t, int token,
                                                int key0) {
  const int32_t *mine = p.masks + (int64_t)token * p.mask_stride;
  const int first = (key0 - t.base) >> 5;
  TreeWords x;
#pragma unroll
  for (int i = 0; i <= KEYS / 32; ++i) {
    const int at = first + i, last = p.words - 1;
    const uint32_t word = (uint32_t)mine[at < 0 ? 0 : at < last ? at : last];
    x.w[i] = at < 0 || at > last ? ~0u : word;
  }
  return x;
}
__device__ __forceinline__ uint32_t tree_bits(const PagedTile &t,
                                              const TreeWords &x, int key0,
                                              int half) {
  return __builtin_amdgcn_alignbit(x.w[half + 1], x.w[half],
                                   (uint32_t)(key0 - t.base) & 31);
}

// The packed row of the small requests' row r: the last lane whose small rows
// start at or before it, then its requests one after the other. Unsigned, and
// a packed row whatever row_starts hold (the lanes' sums may have wrapped).
template <PagedKeys KIND>
__device__ __forceinline__ int packed_row(const PagedAttention &p,
                                          const Requests &all, uint32_t r) {
  int l = 0;
#pragma unroll
  for (int step = 32; step > 0; step >>= 1)
    if (all.small[l + step] <= r)
      l += step;
  uint32_t rest = r - all.small[l];
  const int each = (p.batch + 63) >> 6;
  int begin = all.of[0][l];
  if (each > 1) {
    int b = l * each;
    const int last = b + each < p.batch ? b + each - 1 : p.batch - 1;
    for (;; ++b) {
      begin = row_start(p, b);
      const int rows = (row_start(p, b + 1) - begin) * p.group;
      const uint32_t mine = rows > 0 && rows <= kSharedRows<KIND> ? rows : 0;
      if (rest < mine || b >= last)
        break;
      rest -= mine;
    }
  }
  r = (uint32_t)(begin * p.group) + rest;
  const uint32_t end = (uint32_t)(p.rows * p.group);
  return (int)(r < end ? r : end - 1);
}

// The lane's query row of a tile.
template <PagedKeys KIND>
__device__ __forceinline__ const f16 *query_row(const PagedAttention &p,
                                                const PagedTile &t,
                                                const Requests &all, int r) {
  if (t.compact)
    r = packed_row<KIND>(p, all, (uint32_t)r);
  const int token = token_of(p, r);
  return p.q + (int64_t)token * p.q_row +
         (int64_t)(t.kv_head * p.group + r - token * p.group) * p.q_head;
}

// Inclusive sums over the lanes.
__device__ __forceinline__ uint32_t lane_sums(uint32_t x) {
#define IHP_SHIFTED(CTRL, ROWS)                                                \
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false)
  IHP_SHIFTED(0x111, 0xf);  // row_shr 1, 2, 4, 8: sums within 16 lanes
  IHP_SHIFTED(0x112, 0xf);
  IHP_SHIFTED(0x114, 0xf);
  IHP_SHIFTED(0x118, 0xf);
  IHP_SHIFTED(0x142, 0xa);  // row_bcast 15: rows 1, 3 take rows 0, 2's
  IHP_SHIFTED(0x143, 0xc);  // row_bcast 31: rows 2, 3 take rows 0 and 1's
#undef IHP_SHIFTED
  return x;
}

// Where a tile's keys are, in scalar registers for the length of its loop.
struct Pages {
  const int32_t *prefix_pages, *table;
  int prefix, own_end;  // keys
  int pages, page_size, shift, near;
  uint32_t magic, k_page, k_row, v_page, v_row, key0;

  __device__ __forceinline__ Pages(const PagedAttention &p, const PagedTile &t)
      : prefix_pages(held(p.prefix_pages)), table(held(t.table)),
        prefix(held(p.prefix)), own_end(held(t.own_end)), pages(held(p.pages)),
        page_size(held(p.page_size)), shift(held(p.page_shift)),
        near(held(p.near)), magic(held(p.page_magic)),
        k_page(held(p.k_page16)), k_row(held(p.k_row16)),
        v_page(held(p.v_page16)), v_row(held(p.v_row16)),
        key0((uint32_t)t.key0) {}
};

// Pages of the KEYS keys of a block: a lane's key, its table's page number
// (find, a block ahead of the rows) and the places in the caches that `place`
// makes of it, in 16 bytes. A page that the cache does not have hides its
// keys.
template <int KEYS, PagedKeys KIND>
struct PagedBlock {
  typedef typename std::conditional<KEYS == 64, uint64_t, uint32_t>::type Mask;
  int found = 0, inside = 0;
  uint32_t k = 0, v = 0;
  Mask there = 0;  // bit i: key i of the block is there

  // `lead`: the prefix's blocks of KEYS keys. Keys past the end are the last
  // one, or those of the last aligned `group` keys (which a page that is a
  // multiple of them holds whole).
  __device__ __forceinline__ void find(const Pages &p, int lead, int c,
                                       int group = 1) {
    if constexpr (KIND == PagedKeys::kRows) {
      const int key = c * KEYS + ((int)threadIdx.x & (KEYS - 1));
      inside = key < p.own_end ? key : p.own_end - 1;
      return;
    }
    const bool own = c >= lead;
    const int end = own ? p.own_end : p.prefix;
    const int32_t *table = own ? p.table : p.prefix_pages;
    int key = (own ? c - lead : c) * KEYS + ((int)threadIdx.x & (KEYS - 1));
    if (key >= end)
      key = ((end - 1) & -group) + (key & (group - 1));
    const int column =
        p.page_size == 1 ? key : (int)(__umulhi((uint32_t)key, p.magic) >> p.shift);
    inside = key - column * p.page_size;
    found = table[column];
  }
  __device__ __forceinline__ void place(const Pages &p, int lead, int c) {
    const bool own = c >= lead;
    const int left = own ? p.own_end - (c - lead) * KEYS : p.prefix - c * KEYS;
    if constexpr (KIND == PagedKeys::kRows) {
      k = (p.key0 + (uint32_t)inside) * p.k_row;
      v = (p.key0 + (uint32_t)inside) * p.v_row;
      there = left < KEYS ? ((Mask)1 << left) - 1 : ~(Mask)0;
      return;
    }
    const bool has = (uint32_t)found < (uint32_t)p.pages;
    const uint32_t page = has ? (uint32_t)found : 0u;
    if (p.near) {  // every factor below 2^24
      k = __umul24(page, p.k_page) + __umul24(inside, p.k_row);
      v = __umul24(page, p.v_page) + __umul24(inside, p.v_row);
    } else {
      k = page * p.k_page + (uint32_t)inside * p.k_row;
      v = page * p.v_page + (uint32_t)inside * p.v_row;
    }
    there = (Mask)__ballot(has);
    if (left < KEYS)
      there = left > 0 ? there & (((Mask)1 << left) - 1) : 0;
  }
};

// Where a row's result or part goes.
__device__ __forceinline__ int64_t result_row(const PagedAttention &p,
                                              int kv_head, int row) {
  const int token = token_of(p, row);
  return (int64_t)token * p.o_row +
         (int64_t)(kv_head * p.group + row - token * p.group) * p.o_head;
}
// Four columns of it.
template <bool F32>
__device__ __forceinline__ void store_result(const PagedAttention &p,
                                             int64_t at, f32x4 x) {
  if (F32)
    *(f32x4 *)((float *)p.o + at) = x;
  else
    *(f16x4 *)(p.o + at) = f16x4{(f16)x[0], (f16)x[1], (f16)x[2], (f16)x[3]};
}
// Two weights 2^(s - m) as the matrix instruction takes them, in f16: rounded by
// at most 2^-11 of each or, the largest being 1, 2^-25; their sum is of the
// rounded ones. That is of the size of an f16 result's own rounding. F32: a
// result of 32 bits gets 22 bits of them, what the rounding leaves as a second
// operand and half as many products again (one prompt of 8191 tokens, 32 / 8 heads
// of 128: 783 us instead of 556, so f16 results do without). Both are 2^11 times
// the weight, which the sums cancel: what neither holds is then 2^-22 of it or
// 2^-36.
struct Weights {
  f16x2 f16s, rest;
};
template <bool F32>
__device__ __forceinline__ Weights weights_of(float x, float y) {
  Weights w = {};
  if constexpr (F32) {
    x *= 2048.0f;
    y *= 2048.0f;
  }
  w.f16s = __builtin_convertvector(f32x2{x, y}, f16x2);
  if constexpr (F32)
    w.rest = f16x2{(f16)(x - (float)w.f16s[0]), (f16)(y - (float)w.f16s[1])};
  return w;
}

__device__ __forceinline__ int64_t part_row(const PagedAttention &p,
                                            const PagedTile &t, int row) {
  return (int64_t)t.kv_head * p.part_rows + t.part + row;
}

}  // namespace

// A tile of up to 16 rows. DP: the row of a staged V (64, 128 or 256); DX: a
// multiple of 32 up to it, at least V's head dim; DK: alike of Q's and K's.
template <int DP, int DX, int DK, PagedKeys KIND, bool F32>
__device__ __forceinline__ void narrow_tile(const PagedTile &t,
                                            const Requests &all, char *smem,
                                            float (*wave_m)[kNarrowRows],
                                            float (*wave_l)[kNarrowRows]) {
  const PagedAttention &p = arguments();
  asm volatile("" ::"s"(p.q), "s"(p.q_row), "s"(p.q_head), "s"(p.k_cache),
               "s"(p.v_cache), "s"(p.k_head), "s"(p.v_head), "s"(p.group),
               "s"(p.group_magic), "s"(p.group_shift), "s"(p.dqk), "s"(p.dv),
               "s"(p.scale), "s"(p.prefix_pages), "s"(p.prefix), "s"(p.pages),
               "s"(p.page_size), "s"(p.page_shift), "s"(p.page_magic),
               "s"(p.near), "s"(p.k_page16), "s"(p.k_row16), "s"(p.v_page16),
               "s"(p.v_row16));
  constexpr int KS = DK / 32;           // head-dim steps of S
  constexpr int DB = DX / 16;           // 16-wide d blocks of O
  constexpr int NCH = DP / 8;           // 16-byte chunks of a V row
  constexpr int VROWS = 64 / NCH;       // V rows per load
  constexpr int VP = kBlockKeys / VROWS;
  constexpr int VBYTES = kBlockKeys * DP * 2;
  constexpr int OPITCH = DP + 4;        // floats, merge rows

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l15 = lane & 15, lg = lane >> 4;
  const char *Kp = (const char *)(p.k_cache + (int64_t)t.kv_head * p.k_head);
  const char *Vp = (const char *)(p.v_cache + (int64_t)t.kv_head * p.v_head);

  // This lane's query row (rows past the end repeat the last one), the own
  // keys that it sees, and those that every row sees.
  const int r_mine = t.r0 + l15 < t.r_end ? t.r0 + l15 : t.r_end - 1;
  const int limit = sees(p, t, r_mine);
  const int all_own = KIND == PagedKeys::kTree ? t.base : sees(p, t, t.r0);
  const int token = token_of(p, r_mine);
  i32x4 qf[KS];
  {
    const f16 *qp = query_row<KIND>(p, t, all, r_mine);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int c = 32 * ks + 8 * lg;
      qf[ks] = i32x4{0, 0, 0, 0};
      if (c < p.dqk)
        qf[ks] = *(const i32x4 *)(qp + c);
    }
  }

  // Chunks of a row past the head dim: K's are zeroed before use, V's reach
  // columns that are not stored; both are loaded from inside the row.
  const bool pad_k = p.dqk != DK;
  int koff[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int c = 32 * ks + 8 * lg;
    koff[ks] = 2 * (c < p.dqk ? c : p.dqk - 8);
  }
  const int vrow = lane / NCH, vch = lane % NCH;
  const int voff = 2 * (8 * vch < p.dv ? 8 * vch : p.dv - 8);

  const int lead = t.lead * (kStepKeys / kBlockKeys);
  const int c_begin = t.s_begin * (kStepKeys / kBlockKeys);
  int c_end = lead + (t.seen + kBlockKeys - 1) / kBlockKeys;
  if (c_end > t.s_end * (kStepKeys / kBlockKeys))
    c_end = t.s_end * (kStepKeys / kBlockKeys);
  const Pages pages(p, t);
  PagedBlock<kBlockKeys, KIND> block;
  // The mask's words of a block, read with its rows.
  TreeWords tree = {{~0u, ~0u, ~0u}}, tree_next = tree;
  auto load_tree = [&](int c) __attribute__((always_inline)) {
    const int key0 = (c - lead) * kBlockKeys;
    if (KIND == PagedKeys::kTree && c >= lead && key0 + kBlockKeys > t.base)
      tree_next = tree_words<kBlockKeys>(p, t, token, key0);
  };
  i32x4 kf[2][KS], vf[VP];
  auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const uint32_t at = (uint32_t)__shfl((int)block.k, f * 16 + l15);
      const char *row = Kp + (uint64_t)at * 16;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        kf[f][ks] = *(const i32x4 *)(row + koff[ks]);
    }
  };
  auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const uint32_t at = (uint32_t)__shfl((int)block.v, i * VROWS + vrow);
      vf[i] = *(const i32x4 *)(Vp + (uint64_t)at * 16 + voff);
    }
  };

  f32x4 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
    o[d] = f32x4{0, 0, 0, 0};
  float m_ref = kNegInf, l_sum = 0.0f;
  char *vs = smem + wave * VBYTES;
  const float scale = p.scale * kLog2e;
  const f16x2 ones = {(f16)1.0f, (f16)1.0f};

  // Every wave has finished with the LDS of the tile before.
  __syncthreads();
  int c = c_begin + wave;
  if (c < c_end) {
    block.find(pages, lead, c);
    block.place(pages, lead, c);
    load_k();
    load_v();
    load_tree(c);
    if (c + kPagedWaves < c_end)
      block.find(pages, lead, c + kPagedWaves);
  }
  for (; c < c_end; c += kPagedWaves) {
    const bool more = c + kPagedWaves < c_end;
    const bool own = c >= lead;
    const int key0 = (own ? c - lead : c) * kBlockKeys;
    const uint32_t live = block.there;
    tree = tree_next;
    if (pad_k) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        if (32 * ks + 8 * lg >= p.dqk)
          kf[0][ks] = kf[1][ks] = i32x4{0, 0, 0, 0};
    }
    f32x4 s[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      s[f] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s[f] = Mfma16<f16>::mma(kf[f][ks], qf[ks], s[f]);
      s[f] *= scale;
    }
    if (live != 0xffffffffu || (own && key0 + kBlockKeys > all_own)) {
      const int end = (own ? limit : pages.prefix) - key0;
      uint32_t seen = live;
      if (KIND == PagedKeys::kTree && own && key0 + kBlockKeys > t.base)
        seen &= tree_bits(t, tree, key0, 0);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = 16 * (e >> 2) + 4 * lg + (e & 3);
        if (key >= end || !(seen >> key & 1))
          s[e >> 2][e & 3] = kNegInf;
      }
    }
    if (more) {
      block.place(pages, lead, c + kPagedWaves);
      load_k();
      load_tree(c + kPagedWaves);
      if (c + 2 * kPagedWaves < c_end)
        block.find(pages, lead, c + 2 * kPagedWaves);
    }

    float top = s[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e)
      top = fmaxf(top, s[e >> 2][e & 3]);
    if (__any(top > m_ref)) {
      const float x = fmaxf(m_ref, across_groups_max(top));
      const float keep =
          x == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m_ref - x);
      m_ref = x;
      l_sum *= keep;
#pragma unroll
      for (int d = 0; d < DB; ++d)
        o[d] *= keep;
    }
    const float ref = m_ref == kNegInf ? 0.0f : m_ref;
    i32x4 pf, pf_rest;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x0 = s[e >> 1][2 * (e & 1)], x1 = s[e >> 1][2 * (e & 1) + 1];
      const Weights w = weights_of<F32>(__builtin_amdgcn_exp2f(x0 - ref),
                                        __builtin_amdgcn_exp2f(x1 - ref));
      l_sum = __builtin_amdgcn_fdot2(w.f16s, ones, l_sum, false);
      pf[e] = __builtin_bit_cast(int, w.f16s);
      if constexpr (F32) {
        l_sum = __builtin_amdgcn_fdot2(w.rest, ones, l_sum, false);
        pf_rest[e] = __builtin_bit_cast(int, w.rest);
      }
    }

    // V through this wave's LDS tile; keys that are not there are zeros.
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const int k = i * VROWS + vrow;
      if (!(live >> k & 1))
        vf[i] = i32x4{0, 0, 0, 0};
      *(i32x4 *)(vs + k * (DP * 2) + ((vch ^ row_v_swizzle<NCH>(k)) << 4)) =
          vf[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (more)
      load_v();
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      const int k = 4 * lg + (l15 >> 2);
      const int byte = 2 * (16 * d + 4 * (l15 & 3));
      const IHP_LDS char *at =
          (const IHP_LDS char *)vs + k * (DP * 2) +
          (((byte >> 4) ^ row_v_swizzle<NCH>(k)) << 4) + (byte & 15);
      const i32x2 lo = __builtin_bit_cast(
          i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((IHP_LDS s16x4 *)at));
      const i32x2 hi = __builtin_bit_cast(
          i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                     (IHP_LDS s16x4 *)(at + 16 * (DP * 2))));
      const i32x4 values = {lo[0], lo[1], hi[0], hi[1]};
      o[d] = Mfma16<f16>::mma(values, pf, o[d]);
      if constexpr (F32)
        o[d] = Mfma16<f16>::mma(values, pf_rest, o[d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // Merge the waves: a common max per row, O scaled to it. A row whose
  // scores are all NaN has m -inf and l NaN, which the sums keep.
  const float l_row = across_groups_sum(l_sum);
  if (lg == 0) {
    wave_m[wave][l15] = m_ref;
    wave_l[wave][l15] = l_row;
  }
  __syncthreads();
  float *om = (float *)smem;
  {
    float top = kNegInf;
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w)
      top = fmaxf(top, wave_m[w][l15]);
    const float f =
        m_ref == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m_ref - top);
#pragma unroll
    for (int d = 0; d < DB; ++d)
      *(f32x4 *)(om + (wave * 16 + l15) * OPITCH + 16 * d + 4 * lg) = o[d] * f;
  }
  __syncthreads();
  // Thread (q, dq): row q, DP / 16 columns from dq.
  constexpr int CPT = DP / 16;
  const int q = tid >> 4, dq = (tid & 15) * CPT;
  const int row = t.r0 + q;
  if (row >= t.r_end)
    return;
  float top = kNegInf, sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kPagedWaves; ++w)
    top = fmaxf(top, wave_m[w][q]);
#pragma unroll
  for (int w = 0; w < kPagedWaves; ++w)
    sum += wave_l[w][q] * (wave_m[w][q] == kNegInf
                               ? 0.0f
                               : __builtin_amdgcn_exp2f(wave_m[w][q] - top));
  f32x4 acc[CPT / 4];
#pragma unroll
  for (int e = 0; e < CPT / 4; ++e) {
    acc[e] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w)
      acc[e] += *(const f32x4 *)(om + (w * 16 + q) * OPITCH + dq + 4 * e);
  }
  if (t.part < 0) {
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    const int64_t dst = result_row(p, t.kv_head, row) + dq;
#pragma unroll
    for (int e = 0; e < CPT / 4; ++e)
      if (dq + 4 * e < p.dv)  // dv is a multiple of 8
        store_result<F32>(p, dst + 4 * e, acc[e] * inv);
  } else {
    const int64_t at = part_row(p, t, row);
#pragma unroll
    for (int e = 0; e < CPT / 4; ++e)
      *(f32x4 *)(p.partials + at * DP + dq + 4 * e) = acc[e];
    if (dq == 0)
      *(f32x2 *)(p.part_ml + 2 * at) = f32x2{top, sum};
  }
}

// A tile of up to 128 rows, 32 a wave: K and V of 64 keys in a two-slot LDS
// ring, rows of 16-byte chunks swizzled on the copy side (as attention.hip's):
// K is read 16 lanes = 16 keys at one chunk, V transposed, 32 lanes = 4 keys
// x 32 columns.
// Elements of a staged K row: V's, or the next power of two.
constexpr int staged_k(int dp, int dk) { return dk > dp ? 2 * dp : dp; }
template <int DP>
__device__ __forceinline__ int wide_k_swizzle(int key) {
  return DP >= 128 ? (key & 15) : ((key >> 1) & 7);
}
template <int DP>
__device__ __forceinline__ int wide_v_swizzle(int key) {
  return DP >= 128 ? 4 * (key & 3) : 4 * ((key >> 1) & 1);
}

template <int DP, int DX, int DK, PagedKeys KIND, bool F32>
__device__ __forceinline__ void wide_tile(const PagedTile &t,
                                          const Requests &all, char *smem) {
  const PagedAttention &p = arguments();
  constexpr int DS = DK / 16;         // 16-wide d steps of S^T = K Q^T
  constexpr int DT = DX / 32;         // 32-row d tiles of O^T
  // Of K, then V: bytes of a staged row, its 16-byte chunks, rows that a copy
  // instruction moves.
  constexpr int KP = staged_k(DP, DK), KROW = KP * 2, ROW = DP * 2;
  constexpr int KCH = KROW / 16, CH = ROW / 16;
  constexpr int KBLK = kStepKeys * KROW, BLK = kStepKeys * ROW;
  constexpr int KROWS = 64 / KCH, ROWS = 64 / CH;
  constexpr int KPASSES = kStepKeys / (kPagedWaves * KROWS);
  constexpr int PASSES = kStepKeys / (kPagedWaves * ROWS);
  // Passes of K after which its swizzle, of 16 rows, is the same again.
  constexpr int TURN = kPagedWaves * KROWS < 16 ? 16 / (kPagedWaves * KROWS) : 1;
  // LDS reads whose waits are counted here, not by the compiler. A read that is
  // still on its way must stay in its registers, so not where there are, or with
  // F32's second operands might be, too few of them.
  constexpr bool OWN_WAITS = DP < 256 && !F32;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, l32 = lane & 31;
  const char *Kp = (const char *)(p.k_cache + (int64_t)t.kv_head * p.k_head);
  const char *Vp = (const char *)(p.v_cache + (int64_t)t.kv_head * p.v_head);

  // This lane's query row (rows past the end repeat the last one) and the own
  // keys that it sees; those that every row of the wave sees.
  const int r_wave = t.r0 + 32 * wave;
  const int r_mine = r_wave + l32 < t.r_end ? r_wave + l32 : t.r_end - 1;
  const bool idle = r_wave >= t.r_end;  // no rows: the wave only copies
  const int limit = sees(p, t, r_mine);
  const int all_own =
      KIND == PagedKeys::kTree
          ? t.base
          : sees(p, t, r_wave < t.r_end ? r_wave : t.r_end - 1);
  const int token = token_of(p, r_mine);

  // Copy side: an instruction moves ROWS rows of CH chunks, lane -> (row,
  // physical chunk), fetching the logical chunk that belongs there if it lies
  // within the head dim (the LDS past it is zeroed once and never written).
  // The swizzles repeat every 16 rows, so V's chunk is the same in all passes.
  // Where pages are multiples of ROWS tokens an instruction's rows follow one
  // another in a page; with a head's rows within 4 GiB their place is then one
  // scalar offset, and a lane's own the same for all copies: 28 instructions a
  // block instead of 100 (four prompts of 2243 rows 255.7 -> 247.3 us on one
  // card, others the same).
  static_assert(ROWS % KROWS == 0, "a group of V's rows holds K's");
  const int k_at = lane / KCH, v_at = lane / CH;
  int k_chunk[TURN];
  bool k_in[TURN];
#pragma unroll
  for (int i = 0; i < TURN; ++i) {
    k_chunk[i] = lane % KCH ^ wide_k_swizzle<KP>(
                                  (i * kPagedWaves + wave) * KROWS + k_at);
    k_in[i] = 8 * k_chunk[i] < p.dqk;
  }
  const int v_chunk = lane % CH ^ wide_v_swizzle<DP>(wave * ROWS + v_at);
  const bool v_in = 8 * v_chunk < p.dv;
  const Pages pages(p, t);
  const bool grouped = KIND != PagedKeys::kRows && pages.near &&
                       pages.page_size % ROWS == 0;
  const bool alike = KPASSES == PASSES && pages.k_page == pages.v_page &&
                     pages.k_row == pages.v_row;
  const int group = grouped ? ROWS : 1;
  uint32_t k_lane[TURN];
#pragma unroll
  for (int i = 0; i < TURN; ++i)
    k_lane[i] = ((uint32_t)k_at * pages.k_row + k_chunk[i]) * 16;
  const uint32_t v_lane = ((uint32_t)v_at * pages.v_row + v_chunk) * 16;
  const i32x4 k_rows = rows_from(Kp), v_rows = rows_from(Vp);
  IHP_LDS char *lds = (IHP_LDS char *)smem;
  PagedBlock<kStepKeys, KIND> block;
  // kRows: a whole block's rows follow one another, so its place is the
  // descriptor's base, a pass of the copy a scalar offset and a lane's own the
  // same for all. The last keys, fewer than a block, take the others' way.
  const char *Kq = Kp + t.key0 * pages.k_row * 16;
  const char *Vq = Vp + t.key0 * pages.v_row * 16;
  auto copy_rows = [&](int slot, int key0) {
    IHP_LDS char *kd = lds + slot * KBLK + wave * (KROWS * KROW);
    IHP_LDS char *vd = lds + 2 * KBLK + slot * BLK + wave * (ROWS * ROW);
    constexpr int KNEXT = kPagedWaves * KROWS * KROW;
    constexpr int NEXT = kPagedWaves * ROWS * ROW;
    const i32x4 kr = rows_from(Kq + (int64_t)key0 * (pages.k_row * 16));
    const i32x4 vr = rows_from(Vq + (int64_t)key0 * (pages.v_row * 16));
#pragma unroll
    for (int turn = 0; turn < TURN; ++turn)
      if (k_in[turn])
#pragma unroll
        for (int i = turn; i < KPASSES; i += TURN)
          buffer_to_lds_16(kr, k_lane[turn],
                           (uint32_t)(i * kPagedWaves + wave) *
                               (KROWS * 16 * pages.k_row),
                           kd + i * KNEXT);
    if (v_in)
#pragma unroll
      for (int i = 0; i < PASSES; ++i)
        buffer_to_lds_16(vr, v_lane,
                         (uint32_t)(i * kPagedWaves + wave) *
                             (ROWS * 16 * pages.v_row),
                         vd + i * NEXT);
  };
  auto copy = [&](int slot) {
    IHP_LDS char *kd = lds + slot * KBLK + wave * (KROWS * KROW);
    IHP_LDS char *vd = lds + 2 * KBLK + slot * BLK + wave * (ROWS * ROW);
    constexpr int KNEXT = kPagedWaves * KROWS * KROW;
    constexpr int NEXT = kPagedWaves * ROWS * ROW;
    if (grouped) {
      uint32_t at[KPASSES];
#pragma unroll
      for (int i = 0; i < KPASSES; ++i)
        at[i] = (uint32_t)__builtin_amdgcn_readlane(
                    (int)block.k, (i * kPagedWaves + wave) * KROWS) *
                16;
#pragma unroll
      for (int turn = 0; turn < TURN; ++turn)
        if (k_in[turn])
#pragma unroll
          for (int i = turn; i < KPASSES; i += TURN)
            buffer_to_lds_16(k_rows, k_lane[turn], at[i], kd + i * KNEXT);
      if (!alike)
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
          at[i] = (uint32_t)__builtin_amdgcn_readlane(
                      (int)block.v, (i * kPagedWaves + wave) * ROWS) *
                  16;
      if (v_in)
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
          buffer_to_lds_16(v_rows, v_lane, at[i], vd + i * NEXT);
    } else {
      uint32_t k_of[KPASSES], v_of[PASSES];
#pragma unroll
      for (int i = 0; i < KPASSES; ++i)
        k_of[i] = (uint32_t)__shfl(
            (int)block.k, (i * kPagedWaves + wave) * KROWS + k_at);
#pragma unroll
      for (int i = 0; i < PASSES; ++i)
        v_of[i] = (uint32_t)__shfl(
            (int)block.v, (i * kPagedWaves + wave) * ROWS + v_at);
#pragma unroll
      for (int turn = 0; turn < TURN; ++turn)
        if (k_in[turn])
#pragma unroll
          for (int i = turn; i < KPASSES; i += TURN)
            global_to_lds_16(
                Kp + ((uint64_t)k_of[i] + (uint32_t)k_chunk[turn]) * 16,
                kd + i * KNEXT);
      if (v_in)
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
          global_to_lds_16(Vp + ((uint64_t)v_of[i] + (uint32_t)v_chunk) * 16,
                           vd + i * NEXT);
    }
  };

  // K read base of this lane in slot 0; a d step's address is it XOR 32 s (the
  // ring is aligned, and the swizzle flips chunk bits only). V^T reads: load
  // lane j = lane % 16 of block b = lane / 16 reads row kstart + j / 4,
  // columns 32 dt + 16 (b % 2) + 4 (j % 4) .. + 3.
  const int k_sw = wide_k_swizzle<KP>(l32);
  const uint32_t ka =
      (uint32_t)(uintptr_t)lds +
      (uint32_t)(l32 * KROW + 16 * (g ^ (k_sw & 1)) + 32 * (k_sw >> 1));
  const int vj = lane & 15, vb = lane >> 4;
  int v_off[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const int b0 = 64 * dt + 2 * (16 * (vb & 1) + 4 * (vj & 3));
    v_off[dt] = (4 * g + (vj >> 2)) * ROW +
                (((b0 >> 4) ^ wide_v_swizzle<DP>(vj >> 2)) << 4) + (b0 & 15);
  }

  f32x16 o[DT], st[2];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    o[dt] = f32x16{};
  float m_run = kNegInf, l_run = 0.0f;  // l_run: this lane half's keys
  const float scale = p.scale * kLog2e;

  const int lead = t.lead;
  int c_end = lead + (t.seen + kStepKeys - 1) / kStepKeys;
  if (c_end > t.s_end)
    c_end = t.s_end;
  int c = t.s_begin;
  // Every wave has finished with the LDS of the tile before.
  wait_lgkmcnt0();
  block_barrier();
  if (p.dqk != DK || p.dv != DX) {
    for (int i = tid * 16; i < 2 * (KBLK + BLK); i += kPagedThreads * 16)
      *(IHP_LDS i32x4 *)(lds + i) = i32x4{0, 0, 0, 0};
    wait_lgkmcnt0();
    block_barrier();
  }
  // Block n's rows into a slot.
  auto fetch = [&](int n, int slot) {
    if (KIND == PagedKeys::kRows && (n + 1) * kStepKeys <= pages.own_end) {
      block.there = ~0ull;
      copy_rows(slot, n * kStepKeys);
      return;
    }
    if (KIND == PagedKeys::kRows)
      block.find(pages, lead, n);
    block.place(pages, lead, n);
    copy(slot);
  };
  if (c < c_end) {
    if (KIND != PagedKeys::kRows)
      block.find(pages, lead, c, group);
    fetch(c, 0);
    if (KIND != PagedKeys::kRows && c + 1 < c_end)
      block.find(pages, lead, c + 1, group);
  }
  // The query rows, read while the first keys are.
  i32x4 qf[DS];
  {
    const f16 *qp = query_row<KIND>(p, t, all, r_mine);
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      const int d = 16 * s + 8 * g;
      qf[s] = i32x4{0, 0, 0, 0};
      if (d < p.dqk)
        qf[s] = *(const i32x4 *)(qp + d);
    }
    // Waited for here, or the compiler would at their use in every step.
    wait_vmcnt<0>();
#pragma unroll
    for (int s = 0; s < DS; ++s)
      lgkm_tie(qf[s]);
  }
  for (int slot = 0; c < c_end; ++c, slot ^= 1) {
    const bool own = c >= lead;
    const int key0 = (own ? c - lead : c) * kStepKeys;
    const uint64_t live = block.there;
    // This block's rows have landed, and every wave is done with the one
    // before, whose slot the next one takes.
    wait_vmcnt<0>();
    block_barrier();
    if (live != ~0ull) {  // keys that are not there: their V rows are zeros
      for (int i = tid; i < kStepKeys * CH; i += kPagedThreads)
        if (!(live >> (i / CH) & 1))
          *(IHP_LDS i32x4 *)(lds + 2 * KBLK + slot * BLK + i * 16) =
              i32x4{0, 0, 0, 0};
      wait_lgkmcnt0();
      block_barrier();
    }
    if (c + 1 < c_end) {
      fetch(c + 1, slot ^ 1);
      if (KIND != PagedKeys::kRows && c + 2 < c_end)
        block.find(pages, lead, c + 2, group);
    }

    if (idle)
      continue;

    // S^T: reads run three MFMAs ahead in four rotating registers. The other
    // workgroup's wave on the SIMD leaves its softmax for these.
    __builtin_amdgcn_s_setprio(1);
    {
      const uint32_t kbase = ka + (uint32_t)(slot * KBLK);
      constexpr int NR = 2 * DS, KW = 3, NB = KW + 1;
      i32x4 kb[NB];
      auto issue = [&](auto r_c) {
        constexpr int R = decltype(r_c)::value;
        const IHP_LDS char *at =
            (const IHP_LDS char *)(uintptr_t)(kbase ^ (32u * (R / 2)));
        if constexpr (OWN_WAITS)
          kb[R % NB] = lds_read_16_async<32 * (R % 2) * KROW>(at);
        else
          kb[R % NB] = lds_read_16(at + 32 * (R % 2) * KROW);
      };
      static_for<KW>(issue);
      static_for<NR>([&](auto r_c) {
        constexpr int R = decltype(r_c)::value;
        constexpr int S = R / 2, T = R % 2;
        constexpr int AHEAD = (R + KW < NR ? R + KW : NR) - R - 1;
        if constexpr (OWN_WAITS) {
          lgkm_wait<AHEAD>();
          lgkm_tie(kb[R % NB]);
        }
        st[T] = Mfma32<f16>::mma(kb[R % NB], qf[S], S == 0 ? f32x16{} : st[T]);
        if constexpr (R + KW < NR)
          issue(std::integral_constant<int, R + KW>());
      });
    }

    __builtin_amdgcn_s_setprio(0);

    // Softmax. Element (h, r) of S^T is key 32 h + 8 (r / 4) + 4 g + r % 4.
    float sc = scale;
    if (live != ~0ull || (own && key0 + kStepKeys > all_own) || scale <= 0.0f) {
      const int sees_to = (own ? limit : pages.prefix) - key0;
      uint64_t seen = sees_to >= kStepKeys ? live
                      : sees_to > 0 ? live & ((1ull << sees_to) - 1)
                                    : 0;
      if (KIND == PagedKeys::kTree && own && key0 + kStepKeys > t.base) {
        const TreeWords x = tree_words<kStepKeys>(p, t, token, key0);
        seen &= tree_bits(t, x, key0, 0) |
                (uint64_t)tree_bits(t, x, key0, 1) << 32;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t mine = (uint32_t)(seen >> (32 * h)) >> (4 * g);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          st[h][r] = mine >> (8 * (r >> 2) + (r & 3)) & 1 ? st[h][r] * scale
                                                         : kNegInf;
      }
      sc = 1.0f;
    }
    float top[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top[i] = kNegInf;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        top[i] = fmaxf(top[i], st[i >> 1][8 * (i & 1) + e]);
    }
    const float mx =
        pair_max(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * sc);
    if (!__all(mx <= m_run + kLag)) {
      const float m_new = fmaxf(m_run, mx);
      const float keep =
          m_new == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= keep;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        o[dt] *= keep;
    }
    const float m_use = m_run == kNegInf ? 0.0f : m_run;
    i32x4 pw[4], pw_rest[4];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float p0 = __builtin_amdgcn_exp2f(
            __builtin_fmaf(st[f >> 1][8 * (f & 1) + 2 * w], sc, -m_use));
        const float p1 = __builtin_amdgcn_exp2f(
            __builtin_fmaf(st[f >> 1][8 * (f & 1) + 2 * w + 1], sc, -m_use));
        const Weights x = weights_of<F32>(p0, p1);
        pw[f][w] = __builtin_bit_cast(int, x.f16s);
        if constexpr (F32)
          pw_rest[f][w] = __builtin_bit_cast(int, x.rest);
      }

    // O^T += V^T P^T, 16 keys an MFMA; the V^T fragments of the next key step
    // are read before the MFMAs of this one.
    __builtin_amdgcn_s_setprio(1);
    {
      float psum[4];
      const IHP_LDS char *vs = lds + 2 * KBLK + slot * BLK;
      i32x2 vr[2][DT][2];
      auto read_v = [&](auto step_c) {
        constexpr int ST = decltype(step_c)::value;
        constexpr int KOFF = 16 * ST * ROW;
        static_for<DT>([&](auto dt) {
          constexpr int DTI = decltype(dt)::value;
          if constexpr (OWN_WAITS) {
            vr[ST % 2][DTI][0] = lds_read_tr16_at<KOFF>(vs + v_off[DTI]);
            vr[ST % 2][DTI][1] =
                lds_read_tr16_at<KOFF + 8 * ROW>(vs + v_off[DTI]);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              vr[ST % 2][DTI][i] = __builtin_bit_cast(
                  i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                             (IHP_LDS i16x4 *)(vs + v_off[DTI] + KOFF +
                                               i * 8 * ROW)));
          }
        });
      };
      read_v(std::integral_constant<int, 0>());
      static_for<4>([&](auto step_c) {
        constexpr int ST = decltype(step_c)::value;
        if constexpr (ST < 3)
          read_v(std::integral_constant<int, ST + 1>());
        if constexpr (OWN_WAITS)
          lgkm_wait<ST < 3 ? 2 * DT : 0>();
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          if constexpr (OWN_WAITS) {
            tie2(vr[ST % 2][dt][0]);
            tie2(vr[ST % 2][dt][1]);
          }
          const i32x4 vf = i32x4{vr[ST % 2][dt][0][0], vr[ST % 2][dt][0][1],
                                 vr[ST % 2][dt][1][0], vr[ST % 2][dt][1][1]};
          o[dt] = Mfma32<f16>::mma(vf, pw[ST], o[dt]);
          if constexpr (F32)
            o[dt] = Mfma32<f16>::mma(vf, pw_rest[ST], o[dt]);
        }
        psum[ST] = 0.0f;
        auto add = [&](int two) {
          psum[ST] = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, two),
                                            f16x2{1, 1}, psum[ST], false);
        };
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          add(pw[ST][w]);
          if constexpr (F32)
            add(pw_rest[ST][w]);
        }
      });
      l_run += (psum[0] + psum[1]) + (psum[2] + psum[3]);
    }
    __builtin_amdgcn_s_setprio(0);
  }

  // Register quarter (dt, q) of O^T holds columns 32 dt + 8 q + 4 g .. + 3 of
  // the lane's row.
  const float sum = pair_sum(l_run);
  const int row = r_wave + l32;
  if (KIND != PagedKeys::kPages && !F32 && t.part < 0 && p.o_wide) {
    // The row's lanes exchange halves of two quarters, so that each stores 16
    // bytes of one.
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    f16 *dst = p.o + result_row(p, t.kv_head, row < t.r_end ? row : t.r_end - 1);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; q += 2) {
        i32x4 mine;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 4 * q + 2 * e;
          const f16x2 lo = {(f16)(o[dt][r] * inv), (f16)(o[dt][r + 1] * inv)};
          const f16x2 hi = {(f16)(o[dt][r + 4] * inv),
                            (f16)(o[dt][r + 5] * inv)};
          int a = __builtin_bit_cast(int, lo), b = __builtin_bit_cast(int, hi);
          half_exchange(a, b);
          mine[e] = a;
          mine[2 + e] = b;
        }
        const int d = 32 * dt + 8 * (q + g);
        if (row < t.r_end && d < p.dv)
          *(i32x4 *)(dst + d) = mine;
      }
    return;
  }
  if (row >= t.r_end)
    return;
  if (t.part < 0) {
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    const int64_t dst = result_row(p, t.kv_head, row) + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (32 * dt + 8 * q < p.dv)  // dv is a multiple of 8
          store_result<F32>(
              p, dst + 32 * dt + 8 * q,
              f32x4{o[dt][4 * q] * inv, o[dt][4 * q + 1] * inv,
                    o[dt][4 * q + 2] * inv, o[dt][4 * q + 3] * inv});
  } else {
    const int64_t at = part_row(p, t, row);
    float *dst = p.partials + at * DP + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(f32x4 *)(dst + 32 * dt + 8 * q) =
            f32x4{o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2],
                  o[dt][4 * q + 3]};
    if (g == 0)
      *(f32x2 *)(p.part_ml + 2 * at) = f32x2{m_run, sum};
  }
}

// ----------------------------------------------------------------------------
// The line of a KV head's tiles.
// ----------------------------------------------------------------------------

namespace {

// What keys cost a tile, and back: a wide tile's step is the longer one.
__device__ __forceinline__ uint32_t cost_of(uint32_t keys, int shift) {
  return shift > 4 ? keys + (keys * (kWideCost - 8) >> 3) : keys;
}
__device__ __forceinline__ uint32_t keys_of(uint32_t cost, int shift) {
  return shift > 4 ? cost / kWideCost * 8 + cost % kWideCost * 8 / kWideCost
                   : cost;
}

// Request b's tiles on the line: tile i takes a + i * step units, near the keys
// that it walks and what a tile costs besides, so that their sums have a
// closed form. A unit is 2^unit keys, which keeps the line below 2^31.
struct Request {
  int begin, end, shift, tiles;  // rows' tokens, log2 of a tile's rows
  int own_end, base;
  uint32_t a, step;
  __device__ __forceinline__ uint32_t before(uint32_t i) const {
    return i * a + step * (i * (i - 1) / 2);
  }
};
// A workgroup's place on the line.
struct Line {
  uint32_t x, x_end, start, per;
  float inv_per;
  int kv_head, way, b, i, small_rows;
  bool shared;
  Request q;
};

__device__ __forceinline__ int rows_of(const PagedAttention &p, int begin,
                                       int end) {
  return end > begin ? (end - begin) * p.group : 0;
}

// kRows: the row of request b's first key, and its keys, within the rows that
// there are whatever the starts hold; otherwise its length.
__device__ __forceinline__ int key_start(const PagedAttention &p, int b) {
  const int r = p.lengths[b];
  return r < 0 ? 0 : r > p.key_rows ? p.key_rows : r;
}
template <PagedKeys KIND>
__device__ __forceinline__ int length_of(const PagedAttention &p, int b) {
  if constexpr (KIND == PagedKeys::kRows) {
    const int n = key_start(p, b + 1) - key_start(p, b);
    return n > 0 ? n : 0;
  }
  return p.lengths[b];
}

// `shared`: requests of few rows leave the prefix to tiles of their own.
template <bool WIDE, PagedKeys KIND>
__device__ __forceinline__ Request request(const PagedAttention &p, int begin,
                                           int end, int length, bool shared,
                                           int prefix_keys) {
  Request q;
  const int rows = rows_of(p, begin, end);
  const int added = end > begin ? end - begin : 0;
  const bool small = rows <= kNarrowRows;
  q.begin = begin;
  q.end = begin + added;
  q.shift = !WIDE || small ? 4 : 7;
  q.tiles = (rows + (1 << q.shift) - 1) >> q.shift;
  length = length > 0 ? length : 0;
  q.own_end = length < p.capacity ? length : p.capacity;
  q.base = length - added;
  if (KIND == PagedKeys::kRows && !p.causal)
    q.base = length;  // every row sees them all
  const int tokens =
      small ? added : WIDE ? p.wide_tokens : p.narrow_tokens;
  const bool whole = q.base >= 0 && length <= p.capacity && tokens > 0;
  const bool apart = shared && rows <= kSharedRows<KIND>;
  const uint32_t keys = (uint32_t)(apart ? 0 : prefix_keys) +
                        (uint32_t)(whole ? q.base + tokens : q.own_end);
  q.a = cost_of(keys >> p.unit, q.shift) + p.tile_units;
  if (KIND == PagedKeys::kRows && !p.causal) {
    q.a = cost_of((uint32_t)q.own_end >> p.unit, q.shift) + p.tile_units;
    q.step = 0;
    return q;
  }
  q.step =
      whole && q.tiles > 1 ? cost_of((uint32_t)tokens >> p.unit, q.shift) : 0;
  return q;
}

}  // namespace

// LDS of a tile: a narrow one's V and the waves' merge, a wide one's ring.
constexpr int tile_bytes(int dp, int dk, bool wide) {
  const int v = kPagedWaves * kBlockKeys * dp * 2;
  const int merge = kPagedWaves * 16 * (dp + 4) * 4;
  const int ring = wide ? 4 * kStepKeys * (dp + staged_k(dp, dk)) : 0;
  return ring > v && ring > merge ? ring : v > merge ? v : merge;
}

// WIDE: requests of more than 16 rows have wide tiles. F32: o is (kRows).
template <int DP, int DX, int DK, bool WIDE, PagedKeys KIND, bool F32 = false>
__global__ __launch_bounds__(
    kPagedThreads, DP >= 256 || (WIDE && DK > 128) ? 1 : 2) void
attention_paged_kernel(PagedAttention) {
  __shared__ __attribute__((aligned(1024))) char smem[tile_bytes(DP, DK, WIDE)];
  __shared__ float wave_m[kPagedWaves][kNarrowRows],
      wave_l[kPagedWaves][kNarrowRows];
  // Where each wave is on the line, kept here, out of the tiles' registers.
  // (Every wave finds the same; the requests' are written by all alike.)
  __shared__ Line line_at[kPagedWaves];
  __shared__ Requests all;

  const PagedAttention &p = arguments();
  // What the place on the line takes, in one go instead of each where it is
  // used, a wait apiece (of the other cache lines, a word).
  asm volatile("" ::"s"(p.row_starts), "s"(p.lengths), "s"(p.batch),
               "s"(p.rows), "s"(p.group), "s"(p.prefix), "s"(p.capacity),
               "s"(p.ways), "s"(p.ways_magic), "s"(p.least), "s"(p.unit),
               "s"(p.tile_units), "s"(p.shared), "s"(p.wide_tokens),
               "s"(p.items), "s"(p.table_stride), "s"(p.q_row), "s"(p.k_head));
  // Lane l has requests l * each .. + each - 1.
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int each = (p.batch + 63) >> 6;
  int begin = 0, end = 0, length = 0, key0 = 0;
  if (KIND == PagedKeys::kRows && lane * each < p.batch)
    key0 = key_start(p, lane * each);
  if (lane * each < p.batch) {
    begin = row_start(p, lane * each);
    end = row_start(p, lane * each + 1);
    length = length_of<KIND>(p, lane * each);
  }
  // Consecutive stretches of one head's line read the same prefix: one XCD's.
  int item, unused;
  xcd_tile_order((int)blockIdx.x, p.items, p.items, 1, 1, &item, &unused);
  PagedTile t;
  t.kv_head = p.ways == 1 ? item
                          : (int)__umulhi((uint32_t)item, p.ways_magic);
  int way = item - t.kv_head * p.ways;

  // The small requests' rows, and whether the prefix gets tiles of them.
  auto rest_of_lane = [&](auto f) {  // the lane's requests after its first
    for (int i = 1; i < each && lane * each + i < p.batch; ++i) {
      const int b = lane * each + i;
      f(row_start(p, b), row_start(p, b + 1), length_of<KIND>(p, b));
    }
  };
  auto small_of = [&](int from, int to) {
    const int rows = rows_of(p, from, to);
    return (uint32_t)(rows <= kSharedRows<KIND> ? rows : 0);
  };
  uint32_t small = small_of(begin, end), largest = small;
  rest_of_lane([&](int from, int to, int) {
    const uint32_t n = small_of(from, to);
    small += n;
    largest = n > largest ? n : largest;
  });
  const uint32_t small_upto = lane_sums(small);
  // At most the packed rows, which the parts have room for: requests whose
  // starts do not ascend may count a row several times.
  const uint32_t small_all =
      (uint32_t)__builtin_amdgcn_readlane((int)small_upto, 63);
  const uint32_t rows_all = (uint32_t)(p.rows * p.group);
  int small_rows = (int)(small_all < rows_all ? small_all : rows_all);
  all.of[0][lane] = begin;
  all.of[1][lane] = end;
  all.of[2][lane] = length;
  if (KIND == PagedKeys::kRows)
    all.of[3][lane] = key0;
  all.small[lane] = small_upto - small;
  // shared by two at least: no request has all the small ones' rows
  bool shared = p.shared && small_rows > 0 && !__any(largest == small_all);

  // The line: the prefix's tiles, then the requests'.
  const int prefix_steps = (p.prefix + kStepKeys - 1) / kStepKeys;
  const int prefix_keys = prefix_steps * kStepKeys;
  uint32_t mine;
  {
    const Request q = request<WIDE, KIND>(p, begin, end, length, shared, prefix_keys);
    mine = q.before(q.tiles);
  }
  rest_of_lane([&](int from, int to, int n) {
    const Request q = request<WIDE, KIND>(p, from, to, n, shared, prefix_keys);
    mine += q.before(q.tiles);
  });
  const uint32_t upto = lane_sums(mine);
  Request q = {};
  q.shift = !WIDE || small_rows <= kNarrowRows ? 4 : 7;
  q.tiles = shared ? (small_rows + (1 << q.shift) - 1) >> q.shift : 0;
  q.a = cost_of((uint32_t)prefix_keys >> p.unit, q.shift) + p.tile_units;
  const uint32_t shared_units = q.before(q.tiles);
  const uint32_t total =
      shared_units + (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  // enough for `ways` of them to reach the end (without tiles x is not below)
  uint32_t per = p.ways == 1 ? total : __umulhi(total - 1, p.ways_magic) + 1;
  per = per < (uint32_t)p.least ? p.least : per;
  float inv_per = 1.0f / (float)per;
  uint32_t x = (uint32_t)way * per;  // below 2^32: `ways` is at most 2^24
  if (x >= total)
    return;
  uint32_t x_end = x + per < total ? x + per : total;

  auto request_at = [&](const PagedAttention &p, int b) {
    int of[3];
    if (p.batch <= 64) {
#pragma unroll
      for (int k = 0; k < 3; ++k)
        of[k] = uniform(all.of[k][b]);
    } else {
      of[0] = uniform(row_start(p, b));
      of[1] = uniform(row_start(p, b + 1));
      of[2] = uniform(length_of<KIND>(p, b));
    }
    return request<WIDE, KIND>(p, of[0], of[1], of[2], shared, prefix_keys);
  };

  // Where the stretch begins: among the prefix's tiles, or in the request that
  // holds it: the last lane whose requests start at or before it, then that
  // lane's one after the other; its tile by bisection.
  int b = -1, i = 0;
  uint32_t start = 0;  // where the tiles of b (or of the prefix) start
  if (x >= shared_units) {
    const int lane_of = uniform(
        63 - __builtin_clzll(
                 __ballot(shared_units + upto - mine <= x) | 1));
    start = shared_units +
            (uint32_t)__builtin_amdgcn_readlane((int)(upto - mine), lane_of);
    b = lane_of * each;
    q = request_at(p, b);
    while (start + q.before(q.tiles) <= x && b + 1 < p.batch) {
      start += q.before(q.tiles);
      q = request_at(p, ++b);
    }
  }
  for (int span = q.tiles; span > 1;) {
    const int half = span / 2;
    const bool past = start + q.before(i + half) <= x;
    i += past ? half : 0;
    span = past ? span - half : half;
  }

  while (x < x_end) {
    const PagedAttention &p = arguments();
    asm volatile("" ::"s"(p.batch), "s"(p.rows), "s"(p.group), "s"(p.prefix),
                 "s"(p.capacity), "s"(p.unit), "s"(p.tile_units), "s"(p.snap),
                 "s"(p.wide_tokens), "s"(p.group_magic), "s"(p.group_shift),
                 "s"(p.table), "s"(p.table_stride), "s"(p.packed),
                 "s"(p.partials), "s"(p.part_of));
    if (i >= q.tiles) {  // on to the next request
      start += q.before(q.tiles);
      if (++b >= p.batch)
        return;
      q = request_at(p, b);
      i = 0;
      continue;
    }
    // Units from .. to - 1 of the `units` that the tile has on the line.
    const bool lead = b < 0;
    const uint32_t at = start + q.before(i), units = q.a + q.step * i;
    uint32_t from = x - at;
    uint32_t to = x_end - at < units ? x_end - at : units;
    x = at + to;
    ++i;
    int first = 0, count = 1;
    if (p.partials) {
      // An end less than `snap` from a tile's first key or from its last one
      // moves there: what a part costs is more than it takes off another.
      const uint32_t early = (uint32_t)(p.tile_units + p.snap);
      const uint32_t late = units - (uint32_t)p.snap;
      auto snapped = [&](uint32_t u) {
        return u < early ? 0 : u > late ? units : u;
      };
      // The workgroups of the tile's first and last keys: quotients that the
      // float is off by one of at most.
      auto way_of = [&](uint32_t u) {
        int w = (int)((float)u * inv_per);
        w -= (uint64_t)w * per > u;
        return w + ((uint64_t)(w + 1) * per <= u);
      };
      const uint32_t lead_in = (early < units ? early : units) - 1;
      first = uniform(way_of(at + lead_in));
      count =
          uniform(way_of(at + (late > lead_in ? late : lead_in))) - first + 1;
      from = snapped(from);
      to = to < units ? snapped(to) : units;
      if (from >= to)
        continue;
    } else {
      // without a workspace a workgroup takes the tiles that start in its
      // stretch, whole
      if (from > 0)
        continue;
      to = units;
    }
    t.compact = lead;
    t.r0 = q.begin * p.group + ((i - 1) << q.shift);
    t.r_end = lead ? small_rows : q.end * p.group;
    t.r_end = t.r_end - t.r0 < 1 << q.shift ? t.r_end : t.r0 + (1 << q.shift);
    t.first = q.begin;
    t.base = q.base;
    t.own_end = q.own_end;
    t.table = p.table + (int64_t)(lead ? 0 : b) * p.table_stride;
    t.key0 = 0;
    if (KIND == PagedKeys::kRows)
      t.key0 = uniform(p.batch <= 64 ? all.of[3][b] : key_start(p, b));
    // Whether the tile has all of its rows' keys.
    const bool all_keys =
        !lead && !(shared && (q.end - q.begin) * p.group <= kSharedRows<KIND>);
    t.lead = lead || all_keys ? (p.prefix + kStepKeys - 1) / kStepKeys : 0;
    t.seen = lead ? 0 : uniform(sees(p, t, t.r_end - 1));
    const int steps = t.lead + (t.seen + kStepKeys - 1) / kStepKeys;
    // A tile's own units come first, before its keys.
    auto step_at = [&](uint32_t u) {
      const uint32_t n = keys_of(
          u > (uint32_t)p.tile_units ? u - p.tile_units : 0, q.shift);
      const uint64_t s = (((uint64_t)n << p.unit) + kStepKeys - 1) / kStepKeys;
      return u >= units || s > (uint64_t)steps ? steps : (int)s;
    };
    t.s_begin = step_at(from);
    t.s_end = step_at(to);
    const bool whole = count == 1 && all_keys;
    // kRows has parts of one kind alone.
    const int64_t line = lead || KIND == PagedKeys::kRows ? 0 : p.packed;
    t.part = whole ? -1 : line + (int64_t)kWideRows * way;
    if (p.partials && way == first && t.kv_head == 0)
      for (int r = t.r0 + (int)threadIdx.x; r < t.r_end; r += kPagedThreads) {
        const i32x2 parts = {(int)(line + r) + kWideRows * first,
                             whole ? 0 : count};
        const int at_row = lead ? packed_row<KIND>(p, all, (uint32_t)r) : r;
        p.part_of[line + at_row] = parts;
        if (all_keys)
          p.part_of[p.packed - line + r] = i32x2{0, 0};
      }
    const int shift = q.shift;
    line_at[wave] = {x,  x_end, start, per,        inv_per, t.kv_head,
                     way, b,    i,     small_rows, shared,  q};
    if (shift == 4)
      narrow_tile<DP, DX, DK, KIND, F32>(t, all, smem, wave_m, wave_l);
    else if constexpr (WIDE)
      wide_tile<DP, DX, DK, KIND, F32>(t, all, smem);
    asm volatile("" ::: "memory");
    const Line &l = line_at[wave];
    x = (uint32_t)uniform((int)l.x);
    x_end = (uint32_t)uniform((int)l.x_end);
    start = (uint32_t)uniform((int)l.start);
    per = (uint32_t)uniform((int)l.per);
    inv_per =
        __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, l.inv_per)));
    t.kv_head = uniform(l.kv_head);
    way = uniform(l.way);
    b = uniform(l.b);
    i = uniform(l.i);
    small_rows = uniform(l.small_rows);
    shared = uniform((int)l.shared);
    q.begin = uniform(l.q.begin);
    q.end = uniform(l.q.end);
    q.shift = uniform(l.q.shift);
    q.tiles = uniform(l.q.tiles);
    q.own_end = uniform(l.q.own_end);
    q.base = uniform(l.q.base);
    q.a = (uint32_t)uniform((int)l.q.a);
    q.step = (uint32_t)uniform((int)l.q.step);
  }
}

// Whole tiles: up to so many requests their tiles are counted, four a lane; of
// more, which would make every workgroup count long (4096 of 20 to 200 tokens, 12
// heads of 64: 3692 us, searched 930; 1024 337 and 245, 256 the same, 128 32.5 and
// 34.7), row_starts alone tell where they can begin.
constexpr int kScannedRequests = 256;

// Packed rows whose tiles are all whole: a workgroup takes one, found by the
// requests' numbers of tiles alone (as a line of them 1.5 us longer: 48
// sequences of 1 to 500 tokens, 12 heads of 64, 37.7 -> 34.2 us; prompts of 7195
// rows 119.8 -> 115). Tiles of the most keys come first, by 128 keys, among up to
// 64 requests (16 of 10 to 1500 tokens, 9 / 3 heads of 64: 40.5 -> 34.4 us; 8 of
// 100 to 1500, 24 / 8 heads of 96: 68.2 -> 63.6; of equal length the same; finding
// them costs 0.8, so not where all are short); of more requests, those of each
// one's last tokens. Three workgroups a CU of 64 dims, whose registers just allow it: a
// short sequence's tile is mostly waiting, for its place, its first keys and its
// stores (the 48 sequences 44.7 -> 39.1 us).
template <int DP, int DX, int DK, bool WIDE, bool F32>
__global__ __launch_bounds__(kPagedThreads, DP >= 256 || (WIDE && DK > 128) ? 1
                                            : DP == 64                      ? 3
                                                                            : 2)
void attention_packed_kernel(PagedAttention) {
  constexpr PagedKeys KIND = PagedKeys::kRows;
  constexpr int RESIDENT =
      DP >= 256 || (WIDE && DK > 128) ? 1 : DP == 64 ? 3 : 2;
  __shared__ __attribute__((aligned(1024))) char smem[tile_bytes(DP, DK, WIDE)];
  __shared__ float wave_m[kPagedWaves][kNarrowRows],
      wave_l[kPagedWaves][kNarrowRows];
  __shared__ Requests all;  // not used: no tile is compact

  const PagedAttention &p = arguments();
  asm volatile("" ::"s"(p.row_starts), "s"(p.lengths), "s"(p.batch),
               "s"(p.rows), "s"(p.group), "s"(p.ways), "s"(p.items),
               "s"(p.q_row), "s"(p.causal), "s"(p.key_rows));
  const int lane = threadIdx.x & 63;
  const int each = (p.batch + 63) >> 6;
  int begin = 0, end = 0, key0 = 0, key1 = 0;
  if (p.batch <= kScannedRequests && lane * each < p.batch) {
    begin = row_start(p, lane * each);
    end = row_start(p, lane * each + 1);
    key0 = key_start(p, lane * each);
    key1 = key_start(p, lane * each + 1);
  }
  // Heads that fall to the XCDs evenly stay on one, for its L2; of others all
  // heads' tiles of the most keys come first.
  PagedTile t = {};
  int way, wg = (int)blockIdx.x;
  const bool even = p.kv_heads % 8 == 0;
  // Where all run at once the CUs' second workgroups come in the opposite order
  // of the first ones: the CU with the most keys gets the fewest (a prompt of 2000
  // tokens, 32 / 8 heads of 128: 53.3 -> 49.9 us).
  const int turn = wg / kTurnWgs;
  if (p.items <= kTurnWgs * RESIDENT && turn % 2 == 1) {
    const int first = turn * kTurnWgs;
    const int end = p.items < first + kTurnWgs ? p.items : first + kTurnWgs;
    wg = even ? first + end - 8 - wg / 8 * 8 + wg % 8 : first + end - 1 - wg;
  }
  if (even) {
    int item, unused;
    xcd_tile_order(wg, p.items, p.items, 1, 1, &item, &unused);
    t.kv_head = item / p.ways;
    way = item - t.kv_head * p.ways;
  } else {
    way = wg / p.kv_heads;
    t.kv_head = wg - way * p.kv_heads;
  }
  auto tiles_of = [&](int from, int to) {
    const int rows = rows_of(p, from, to);
    const int shift = !WIDE || rows <= kNarrowRows ? 4 : 7;
    return (uint32_t)(rows + (1 << shift) - 1) >> shift;
  };
  auto lane_at = [&](uint32_t first, uint32_t x) {  // the last first <= x
    return uniform(63 - __builtin_clzll(__ballot(first <= x) | 1));
  };
  auto of_lane = [&](uint32_t x, int l) {
    return (uint32_t)__builtin_amdgcn_readlane((int)x, l);
  };
  uint32_t i;
  if (p.batch <= kScannedRequests) {
    const int tiles_rows = rows_of(p, begin, end);
    uint32_t tiles = tiles_of(begin, end);
    for (int i = 1; i < each && lane * each + i < p.batch; ++i)
      tiles += tiles_of(row_start(p, lane * each + i),
                        row_start(p, lane * each + i + 1));
    const uint32_t upto = lane_sums(tiles);
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    if ((uint32_t)way >= total)
      return;
    int lane_of;
    if (p.levels) {
      // Tile `way` of all by their keys, most first: among those of kLevelKeys *
      // level keys and more but not of the next level.
      const uint32_t keys = key1 > key0 ? (uint32_t)(key1 - key0) : 0;
      const int shift = !WIDE || tiles_rows <= kNarrowRows ? 4 : 7;
      auto with = [&](uint32_t level) {  // the request's tiles of so many keys
        const uint32_t least = level * kLevelKeys;
        const uint32_t n =
            p.causal
                ? (uint32_t)((uint64_t)(keys - least) * p.group >> shift) + 1
                : tiles;
        return keys < least ? 0 : n < tiles ? n : tiles;
      };
      uint32_t level = 0;
      for (uint32_t step = (uint32_t)p.levels; step > 0; step >>= 1)
        if (of_lane(lane_sums(with(level + step)), 63) > (uint32_t)way)
          level += step;
      const uint32_t more = with(level + 1);
      const uint32_t mine = (level == 0 ? tiles : with(level)) - more;
      const uint32_t rank =
          (uint32_t)way - of_lane(lane_sums(more), 63);
      const uint32_t before = lane_sums(mine) - mine;
      lane_of = lane_at(before, rank);
      i = of_lane(tiles - 1 - more, lane_of) - (rank - of_lane(before, lane_of));
      if (i >= of_lane(tiles, lane_of))
        return;  // (the sums may have wrapped)
    } else {
      const uint32_t at = total - 1 - (uint32_t)way;
      lane_of = lane_at(upto - tiles, at);
      i = at - of_lane(upto - tiles, lane_of);
    }
    begin = __builtin_amdgcn_readlane(begin, lane_of);
    end = __builtin_amdgcn_readlane(end, lane_of);
    key0 = __builtin_amdgcn_readlane(key0, lane_of);
    key1 = __builtin_amdgcn_readlane(key1, lane_of);
    for (int b = lane_of * each; i >= tiles_of(begin, end);) {
      // (the sums may have wrapped: no further than the last request)
      if (++b >= p.batch)
        return;
      i -= tiles_of(begin, end);
      begin = uniform(row_start(p, b));
      end = uniform(row_start(p, b + 1));
      key0 = uniform(key_start(p, b));
      key1 = uniform(key_start(p, b + 1));
    }
  } else {
    // Request b's tiles are numbered from (whole tiles of rows before it) + b on:
    // always enough, and the numbers past its own are empty. The last request
    // that begins at or before the way's number, by 64ths.
    auto first_tile = [&](int b) {
      return (row_start(p, b) * p.group >> (WIDE ? 7 : 4)) + b;
    };
    const int at = uniform(first_tile(p.batch)) - 1 - way;
    int b = 0;
    for (int span = p.batch; span > 1;) {
      const int step = (span + 63) >> 6, mine = b + lane * step;
      const bool holds = lane * step < span && first_tile(mine) <= at;
      const int from =
          uniform(63 - __builtin_clzll(__ballot(holds) | 1)) * step;
      b += from;
      span = step < span - from ? step : span - from;
    }
    begin = uniform(row_start(p, b));
    end = uniform(row_start(p, b + 1));
    key0 = uniform(key_start(p, b));
    key1 = uniform(key_start(p, b + 1));
    i = (uint32_t)(at - uniform(first_tile(b)));
    if (at < 0 || i >= tiles_of(begin, end))
      return;
  }
  const int rows = rows_of(p, begin, end);
  const int shift = !WIDE || rows <= kNarrowRows ? 4 : 7;
  const int length = key1 > key0 ? key1 - key0 : 0;
  t.key0 = key0;
  t.r0 = begin * p.group + ((int)i << shift);
  t.r_end = begin * p.group + rows;
  t.r_end = t.r_end - t.r0 < 1 << shift ? t.r_end : t.r0 + (1 << shift);
  t.compact = false;
  t.lead = 0;
  t.own_end = length;
  t.first = begin;
  t.base = p.causal ? length - (end - begin) : length;
  t.seen = uniform(sees(p, t, t.r_end - 1));
  t.s_begin = 0;
  t.s_end = (t.seen + kStepKeys - 1) / kStepKeys;
  t.part = -1;
  if (shift == 4)
    narrow_tile<DP, DX, DK, KIND, F32>(t, all, smem, wave_m, wave_l);
  else if constexpr (WIDE)
    wide_tile<DP, DX, DK, KIND, F32>(t, all, smem);
}

// Joins the parts of every row that has some: DP / 4 threads, 4 columns each,
// for every GROUPS-th four of a row's parts, then the GROUPS sums through LDS.
// A row's parts of one kind (the prefix's of a small request, its own or both
// at once) are kWideRows rows apart; part_of tells the first and how many.
template <int DP, int GROUPS, bool F32>
__global__ __launch_bounds__(kPagedThreads) void attention_paged_join_kernel(
    PagedAttention p) {
  constexpr int TPR = DP / 4, ROWS = kPagedThreads / TPR / GROUPS;
  const int tid = threadIdx.x;
  const int g = tid / TPR % GROUPS, dq = 4 * (tid % TPR);
  const uint32_t per_head = ((uint32_t)p.packed + ROWS - 1) / ROWS;
  const int kv_head = (int)(blockIdx.x / per_head);
  const int row =
      (int)(blockIdx.x - kv_head * per_head) * ROWS + tid / (TPR * GROUPS);
  // What part_of holds for a row past the last one is not used, but loaded
  // with the rest.
  const int at = row < (int)p.packed ? row : 0;
  i32x2 of[2] = {p.part_of[at], p.part_of[p.packed + at]};
  const int rows = row_start(p, p.batch);
  asm volatile("" : "+v"(of[0]), "+v"(of[1]));
  const bool real = row < (int)p.packed && row < rows * p.group;
  int from[2], counts[2];
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    // within the head's part rows, whatever it holds
    const int last = (int)p.part_rows - 1;
    from[kind] = of[kind][0] < 0        ? 0
                 : of[kind][0] < last ? of[kind][0]
                                        : last;
    const int most = (last - from[kind]) / kWideRows + 1;
    counts[kind] = of[kind][1] < most ? of[kind][1] : most;
    counts[kind] = real && counts[kind] > 0 ? counts[kind] : 0;
  }
  const int parts = counts[0] + counts[1];
  const int64_t head_at = (int64_t)kv_head * p.part_rows;
  float top = kNegInf, sum = 0.0f;
  f32x4 acc = {0, 0, 0, 0};
  // 4 parts' loads in flight; a part past the last repeats it with weight 0
  for (int s0 = 4 * g; s0 < parts; s0 += 4 * GROUPS) {
    f32x2 ml[4];
    f32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + u < parts ? s0 + u : parts - 1;
      const int64_t i =
          head_at + (s < counts[0] ? from[0] + kWideRows * s
                                   : from[1] + kWideRows * (s - counts[0]));
      ml[u] = *(const f32x2 *)(p.part_ml + 2 * i);
      v[u] = *(const f32x4 *)(p.partials + i * DP + dq);
    }
    asm volatile("" ::"v"(v[1]), "v"(v[2]), "v"(v[3]));
    float x = top;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      x = fmaxf(x, ml[u][0]);
    const float keep = top == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(top - x);
    top = x;
    sum *= keep;
    acc *= keep;
    // A part without a maximum is one whose keys the row does not see (sum 0:
    // left out, an infinite value of a key that others see is none of it) or
    // gives it NaN scores alone (sum NaN: 0 times it stays NaN).
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + u < parts && !(ml[u][0] == kNegInf && ml[u][1] == 0.0f)) {
        const float f = ml[u][0] == kNegInf
                            ? 0.0f
                            : __builtin_amdgcn_exp2f(ml[u][0] - x);
        sum += f * ml[u][1];
        acc += f * v[u];
      }
  }
  if constexpr (GROUPS > 1) {
    __shared__ f32x4 group_acc[kPagedThreads];
    __shared__ f32x2 group_ml[kPagedThreads];
    group_acc[tid] = acc;
    group_ml[tid] = f32x2{top, sum};
    __syncthreads();
    if (g > 0)
      return;
#pragma unroll
    for (int u = 1; u < GROUPS; ++u)
      top = fmaxf(top, group_ml[tid + u * TPR][0]);
    sum = 0.0f;
    acc = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) {
      const f32x2 ml = group_ml[tid + u * TPR];
      const float f =
          ml[0] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml[0] - top);
      sum += f * ml[1];
      acc += f * group_acc[tid + u * TPR];
    }
  }
  // Without parts the workgroup that had the tile whole stored the row.
  if (!real || parts == 0 || dq >= p.dv)
    return;
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  store_result<F32>(p, result_row(p, kv_head, row) + dq, acc * inv);
}

// ----------------------------------------------------------------------------
// Host side.
// ----------------------------------------------------------------------------

namespace {

struct PagedKernel {
  const char *name;
  PagedKeys keys;
  int dp, dx, dk, groups;  // groups: of a joined row's parts
  bool wide, f32;
  const void *fn;
  const void *whole = nullptr;  // where no tile is split
};
const PagedKernel kPagedKernels[] = {
#define IHP_PAGED(NAME, KIND, DP, DX, DK, WIDE, F32)                           \
  {"attention_" NAME, PagedKeys::KIND, DP, DX, DK, 0, WIDE, F32,               \
   (const void *)&attention_paged_kernel<DP, DX, DK, WIDE, PagedKeys::KIND>}
#define IHP_PAGED_ALL(NAME, KIND, F32)                                         \
  IHP_PAGED(NAME "_d64", KIND, 64, 64, 64, true, F32),                         \
      IHP_PAGED(NAME "_d96", KIND, 128, 96, 96, true, F32),                    \
      IHP_PAGED(NAME "_d128", KIND, 128, 128, 128, true, F32),                 \
      IHP_PAGED(NAME "_d192_128", KIND, 128, 128, 192, false, F32),            \
      IHP_PAGED(NAME "_d192_128_rows", KIND, 128, 128, 192, true, F32),        \
      IHP_PAGED(NAME "_d256", KIND, 256, 256, 256, false, F32)
    IHP_PAGED_ALL("paged", kPages, false),
    IHP_PAGED_ALL("tree", kTree, false),
#undef IHP_PAGED
#define IHP_PAGED(NAME, KIND, DP, DX, DK, WIDE, F32)                           \
  {"attention_" NAME, PagedKeys::KIND, DP, DX, DK, 0, WIDE, F32,               \
   (const void *)&attention_paged_kernel<DP, DX, DK, WIDE, PagedKeys::KIND,    \
                                         F32>,                                 \
   (const void *)&attention_packed_kernel<DP, DX, DK, WIDE, F32>}
    IHP_PAGED_ALL("packed", kRows, false),
    IHP_PAGED("packed_d256_rows", kRows, 256, 256, 256, true, false),
    IHP_PAGED_ALL("packed_f32", kRows, true),
    IHP_PAGED("packed_f32_d256_rows", kRows, 256, 256, 256, true, true),
#undef IHP_PAGED_ALL
#undef IHP_PAGED
// The joins are those of all kinds of keys.
#define IHP_JOIN(NAME, DP, GROUPS, F32)                                        \
  {"attention_" NAME "_join_d" #DP "_g" #GROUPS, PagedKeys::kPages, DP, DP,    \
   DP, GROUPS, false, F32,                                                     \
   (const void *)&attention_paged_join_kernel<DP, GROUPS, F32>}
#define IHP_JOIN_ALL(NAME, F32)                                                \
  IHP_JOIN(NAME, 64, 1, F32), IHP_JOIN(NAME, 64, 8, F32),                      \
      IHP_JOIN(NAME, 128, 1, F32), IHP_JOIN(NAME, 128, 8, F32),                \
      IHP_JOIN(NAME, 256, 1, F32), IHP_JOIN(NAME, 256, 4, F32)
    IHP_JOIN_ALL("paged", false),
    IHP_JOIN_ALL("packed_f32", true),
#undef IHP_JOIN_ALL
#undef IHP_JOIN
};
constexpr int kPagedKernelCount =
    sizeof(kPagedKernels) / sizeof(kPagedKernels[0]);

}  // namespace

PagedPlan plan_attention_paged(PagedKeys keys, int64_t rows, int64_t batch,
                               int64_t kv_heads, int64_t group, int64_t prefix,
                               int64_t capacity, int64_t head_dim,
                               int64_t head_dim_v, size_t workspace_limit) {
  PagedPlan p = {};
  const int64_t d = head_dim > head_dim_v ? head_dim : head_dim_v;
  const int64_t packed = rows * group;
  const bool longer_k = d > 128 && head_dim <= 192 && head_dim_v <= 128;
  // Requests that fill wide tiles walk the prefix themselves, as one alone.
  p.shared = prefix > 0 && batch > 1;
  // Wide tiles of longer keys fill a CU's LDS alone: only where some request
  // must have more than 16 rows (653 of two, 3 heads each, 3947 keys ahead:
  // 72.3 -> 38.3 us; 181 rows of 4 heads, 696 ahead: 18.2 -> 21.0), or where
  // narrow tiles of the prefix would read more keys than all requests can have
  // (676 rows of 68 requests, 11936 keys ahead, 740 each at most: 297.8 ->
  // 213.4 us).
  const bool rows_many = packed > batch * kSmallRows;
  const bool prefix_more = p.shared && prefix + capacity > kPagedWholeKeysFew &&
                           packed / kNarrowRows * prefix > batch * capacity;
  const bool packed_keys = keys == PagedKeys::kRows;
  p.wide = d <= 128 || (longer_k && (rows_many || prefix_more)) ||
           (packed_keys && rows_many);
  p.dp = d <= 64 ? 64 : d <= 128 || longer_k ? 128 : 256;
  p.dx = d > 64 && d <= 96 ? 96 : p.dp;
  p.dk = longer_k ? 192 : p.dx;
  const bool two = p.dp < 256 && !(p.wide && p.dk > 128);  // a CU holds
  const int64_t wgs = two ? kPagedTargetWgs : kPagedTargetWgs / 2;
  p.ways = wgs / kv_heads > 1 ? wgs / kv_heads : 1;
  // The line in 32 bits, also where row_starts do not ascend and every request
  // has all rows.
  const int64_t each = packed / (p.wide ? kWideRows : kNarrowRows) + 2;
  const double line = (double)(batch * each + packed) * (kWideCost / 8.0) *
                      (double)(prefix + capacity + rows + 512);
  while (line / (double)((int64_t)1 << p.unit) >= 1e9)
    ++p.unit;
  auto units = [&](int64_t keys) { return (keys >> p.unit) + 1; };
  p.least = units(kPagedLeastKeys);
  p.tile_units = units(kPagedTileKeys);
  p.snap = units(kPagedSnapKeys);
  p.part_rows = (packed_keys ? 1 : 2) * packed + kWideRows * p.ways;
  p.workspace = (int64_t)kWorkspaceCounterBytes + 2 * packed * 8 +
                kv_heads * p.part_rows * (p.dp + 2) * 4;
  const int64_t tiles = batch + packed / (p.wide ? kWideRows : kNarrowRows);
  const int64_t most = tiles * kv_heads > wgs ? kPagedWholeKeys
                       : p.wide && rows_many  ? kPagedWholeKeysWide
                                              : kPagedWholeKeysFew;
  // Packed rows: tiles are split where the longest would keep its workgroup
  // busy for longer than a share of all the work and a second launch take:
  // more than kPackedWholeKeys keys over that share, which grows with the tiles
  // that there are (one prompt of 1024 tokens, 32 / 8 heads of 128, 35.3 -> 28.1
  // us whole, of 2000 61.3 -> 50.0; of 4000, 9 / 3 of 64, 45.4 split, 63.6 whole;
  // one of 2000, 16 heads, 42.2 and 46.3). How long the longest sequence is is not
  // known here: twice the mean is taken.
  const int64_t longest =
      batch > 2 ? 2 * (capacity / batch) : capacity;
  const bool whole =
      longest * (9 * kPagedTargetWgs - 8 * tiles * kv_heads) <=
      kPackedWholeKeys * 9 * kPagedTargetWgs;
  if ((packed_keys ? whole : prefix + capacity <= most) ||
      (uint64_t)p.workspace > workspace_limit || p.part_rows > INT32_MAX) {
    // every tile whole and one unit, so each workgroup takes as many
    p.shared = false;
    p.workspace = p.part_rows = 0;
    p.unit = 31;
    p.least = p.tile_units = p.snap = 1;
    p.ways = 4 * p.ways < tiles && !packed_keys ? 4 * p.ways : tiles;
  }
  return p;
}

hipError_t launch_attention_paged(PagedKeys keys,
                                  const PagedAttention &attention,
                                  const PagedPlan &plan, void *workspace,
                                  void *stream) {
  PagedAttention a = attention;
  a.ways = (int)plan.ways;
  a.items = (int)(plan.ways * a.kv_heads);
  a.least = (int)plan.least;
  a.unit = (int)plan.unit;
  a.tile_units = (int)plan.tile_units;
  // Requests of a lane each that may differ, and more tiles than
  // kPagedTargetWgs, which is what runs at once where a CU holds two workgroups
  // (of 64 dims it holds three, above 128 dims one; the rule is the same).
  a.levels = a.batch > 1 && a.batch <= 64 && a.items > kPagedTargetWgs &&
                     a.key_rows / a.batch >= 2 * (int)kLevelKeys
                 ? 1
                 : 0;
  while (a.levels && (int64_t)a.levels * 2 * (int64_t)kLevelKeys <= a.key_rows)
    a.levels *= 2;
  a.snap = (int)plan.snap;
  a.shared = plan.shared ? 1 : 0;
  // item / ways, exact while item * ways is below 2^32: at most 4 ways to each
  // of 65535 heads, or 2048 workgroups in all (whole tiles of packed rows may be
  // more, and divide); and the ways' share of a line of less than 2^31 units, at
  // most one unit over. (One way's is not used.)
  if (keys != PagedKeys::kRows && (uint64_t)a.items * (uint64_t)a.ways >> 32)
    return hipErrorInvalidValue;
  a.ways_magic = (uint32_t)(((uint64_t)1 << 32) / (uint64_t)plan.ways + 1);
  a.part_rows = plan.part_rows;
  a.part_of = nullptr;
  a.partials = a.part_ml = nullptr;
  const int64_t all = (int64_t)a.kv_heads * a.packed;
  if (plan.workspace) {
    a.partials = (float *)((char *)workspace + kWorkspaceCounterBytes);
    a.part_ml = a.partials + a.kv_heads * plan.part_rows * plan.dp;
    a.part_of = (i32x2 *)(a.part_ml + a.kv_heads * plan.part_rows * 2);
  }
  // Few rows, whose parts can be many: a row's are dealt to groups.
  const bool few =
      all <= (keys == PagedKeys::kPages ? kPagedFewRows : kTreeFewRows);
  const PagedKernel *kernel = nullptr, *join = nullptr;
  for (const PagedKernel &k : kPagedKernels)
    if (k.dp == plan.dp && k.f32 == (a.out_f32 != 0)) {
      if (k.groups == 0 && k.keys == keys && k.dx == plan.dx &&
          k.dk == plan.dk && k.wide == plan.wide)
        kernel = &k;
      else if (k.groups > 0 && (k.groups > 1) == few)
        join = &k;
    }
  if (!kernel || !join)
    return hipErrorInvalidValue;
  void *args[] = {&a};
  const void *fn = !plan.workspace && kernel->whole ? kernel->whole : kernel->fn;
  hipError_t e =
      hipLaunchKernel(fn, dim3((unsigned)a.items),
                      dim3(kPagedThreads), args, 0, (hipStream_t)stream);
  if (e != hipSuccess || !plan.workspace)
    return e;
  const int64_t per = kPagedThreads / (plan.dp / 4) / join->groups;
  const int64_t blocks = (a.packed + per - 1) / per * a.kv_heads;
  return hipLaunchKernel(join->fn, dim3((unsigned)blocks),
                         dim3(kPagedThreads), args, 0, (hipStream_t)stream);
}

const KernelEntry *attention_paged_kernels(int *count) {
  static KernelEntry all[2 * kPagedKernelCount];
  static char names[kPagedKernelCount][48];  // of the whole tiles' kernels
  static const int filled = [] {
    int n = 0;
    for (const PagedKernel &k : kPagedKernels) {
      all[n++] = {k.name, k.fn, kPagedThreads, 0};
      if (k.whole) {
        char *name = names[&k - kPagedKernels];
        snprintf(name, sizeof(names[0]), "%s_whole", k.name);
        all[n++] = {name, k.whole, kPagedThreads, 0};
      }
    }
    return n;
  }();
  *count = filled;
  return all;
}

}  // namespace ihp
