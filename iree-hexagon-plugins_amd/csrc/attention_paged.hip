// Attention over a paged KV cache for a batch whose requests share a prefix.
//
// The new tokens of all requests are packed rows (row_starts); the query rows
// of a KV head are its `group` heads of every token, r = token * group + head.
// A row's keys are the prefix, which every row sees whole, and its request's
// own keys up to itself. Each is a run of pages named by a table. With
//   m = max_j s_j, l = sum_j 2^(s_j - m), a = sum_j 2^(s_j - m) v_j
// of any set of keys (s = q . k * scale * log2 e), two sets join as
//   m = max(m1, m2), l = l1 2^(m1 - m) + l2 2^(m2 - m), a alike, o = a / l,
// so the prefix is computed for tiles of rows of the whole batch, each
// request's own keys for tiles of its own rows, both by key splits, and a
// second kernel joins the parts of each row. Where requests bring enough rows
// to fill tiles, a tile walks the prefix and its own keys in turn and stores
// the result itself.
//
// A workgroup takes a tile of 16 or 32 rows, its 4 waves blocks of 32 keys in
// turn, each alone: K rows go from memory into MFMA fragments (S^T = K Q^T; a
// lane holds 4 + 4 keys of one row), V rows through the wave's LDS tile, from
// which transposed reads take the key order that S^T has, so P stays in
// registers for O^T += V^T P. The next block's rows are in flight during the
// current one, and the page numbers of the one after it.
#include "device_common.h"
#include "kernels_internal.h"

namespace ihp {

namespace {

constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = kPagedThreads / 64;
constexpr int kBlockKeys = 32;
constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;

// Chunk swizzle of a staged V row (key) of NCH 16-byte chunks: a transposed
// read takes 4 rows of one 32-byte window per 16-lane block, two blocks (rows
// 4 apart) at a time, and all of it must spread over the 64 banks.
template <int NCH>
__device__ __forceinline__ int v_swizzle(int k) {
  return NCH >= 16 ? (4 * (k & 3)) ^ (2 * ((k >> 2) & 1))
                   : (2 * ((k >> 1) & 1)) ^ (4 * ((k >> 2) & 1));
}

__device__ __forceinline__ float across_groups_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float across_groups_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// row_starts[b], within the rows that there are whatever it holds.
__device__ __forceinline__ int row_start(const PagedAttention &p, int b) {
  const int r = p.row_starts[b];
  return r < 0 ? 0 : r > p.rows ? p.rows : r;
}

// The request of tile `tile` where request b's tiles of RM rows start at
// row_starts[b] * group / RM + b: at least as many numbers as it has tiles,
// with no sum over the requests. 64 of them are looked at a step.
template <int RM>
__device__ __forceinline__ int request_of(const PagedAttention &p, int tile) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = p.batch;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int b = lo + lane * step;
    const bool at = lane * step < n &&
                    (int64_t)row_start(p, b) * p.group / RM + b <= tile;
    // lanes ascend: the last one that holds
    const int last = 63 - __builtin_clzll(__ballot(at) | 1);
    lo += last * step;
    n = n - last * step < step ? n - last * step : step;
  }
  return lo;
}

}  // namespace

// One tile's work: rows r0 .. r_end - 1 (of a KV head) against key blocks
// c_begin .. c_end - 1, the first `lead` of them the prefix's.
struct PagedTile {
  int kv_head, r0, r_end;
  int lead;            // prefix blocks
  int prefix;          // prefix keys
  const int32_t *table;  // the request's pages
  int own_end;         // own keys that its pages hold
  int base, first;     // row r sees own keys .. base + r / group - first
  int c_begin, c_end;
  int part;            // which part of the rows' keys this is
};

// DP: the head-dim bucket (64, 128 or 256, at least both head dims); RF:
// 16-row fragments a tile.
template <int DP, int RF>
__device__ __forceinline__ void paged_tile(const PagedAttention &p,
                                           const PagedTile &t, char *smem,
                                           float (*wave_m)[32],
                                           float (*wave_l)[32]) {
  constexpr int KS = DP / 32;           // head-dim steps of S
  constexpr int DB = DP / 16;           // 16-wide d blocks of O
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

  // This lane's query rows (rows past the end repeat the last one) and the
  // own keys that they see.
  auto sees = [&](int r) {
    const int64_t n = (int64_t)t.base + r / p.group - t.first + 1;
    return n < 0 ? 0 : n > t.own_end ? t.own_end : (int)n;
  };
  i32x4 qf[RF][KS];
  int limit[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    int r = t.r0 + f * 16 + l15;
    r = r < t.r_end ? r : t.r_end - 1;
    limit[f] = sees(r);
    const f16 *qp = p.q + (int64_t)(r / p.group) * p.q_row +
                    (int64_t)(t.kv_head * p.group + r % p.group) * p.q_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int c = 32 * ks + 8 * lg;
      qf[f][ks] = i32x4{0, 0, 0, 0};
      if (c < p.dqk)
        qf[f][ks] = *(const i32x4 *)(qp + c);
    }
  }
  const int all_own = sees(t.r0);  // own keys that every row sees

  // Chunks of a row past the head dim: K's are zeroed before use, V's reach
  // columns that are not stored; both are loaded from inside the row.
  const bool pad_k = p.dqk != DP;
  int koff[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int c = 32 * ks + 8 * lg;
    koff[ks] = 2 * (c < p.dqk ? c : p.dqk - 8);
  }
  const int vrow = lane / NCH, vch = lane % NCH;
  const int voff = 2 * (8 * vch < p.dv ? 8 * vch : p.dv - 8);

  // Block c's page number and place in it of key lane % 32: loaded (find)
  // one block ahead of the rows, whose places (in 16 bytes) `place` makes of
  // it. A page that the cache does not have hides its keys.
  int found = 0, inside = 0;
  auto find = [&](int c) __attribute__((always_inline)) {
    const bool own = c >= t.lead;
    const int end = own ? t.own_end : t.prefix;
    const int32_t *table = own ? t.table : p.prefix_pages;
    int key = (own ? c - t.lead : c) * kBlockKeys + (lane & 31);
    key = key < end ? key : end - 1;
    const int column =
        (int)(((uint64_t)(uint32_t)key * p.page_magic) >> p.page_shift);
    inside = key - column * p.page_size;
    found = table[column];
  };
  uint32_t kat = 0, vat = 0, there = 0;
  auto place = [&](int c) __attribute__((always_inline)) {
    const bool own = c >= t.lead;
    const int end = own ? t.own_end : t.prefix;
    const int left = end - (own ? c - t.lead : c) * kBlockKeys;
    const bool has = (uint32_t)found < (uint32_t)p.pages;
    const uint32_t page = has ? (uint32_t)found : 0u;
    kat = page * p.k_page16 + (uint32_t)inside * p.k_row16;
    vat = page * p.v_page16 + (uint32_t)inside * p.v_row16;
    there = (uint32_t)__ballot(has);
    if (left < kBlockKeys)
      there &= (1u << left) - 1;
  };

  i32x4 kf[2][KS], vf[VP];
  auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const uint32_t at = (uint32_t)__shfl((int)kat, f * 16 + l15);
      const char *row = Kp + (uint64_t)at * 16;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        kf[f][ks] = *(const i32x4 *)(row + koff[ks]);
    }
  };
  auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const uint32_t at = (uint32_t)__shfl((int)vat, i * VROWS + vrow);
      vf[i] = *(const i32x4 *)(Vp + (uint64_t)at * 16 + voff);
    }
  };

  f32x4 o[RF][DB];
  float m_ref[RF], l_sum[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    m_ref[f] = kNegInf;
    l_sum[f] = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
      o[f][d] = f32x4{0, 0, 0, 0};
  }
  char *vs = smem + wave * VBYTES;
  const float scale = p.scale * kLog2e;
  const f16x2 ones = {(f16)1.0f, (f16)1.0f};

  int c = t.c_begin + wave;
  if (c < t.c_end) {
    find(c);
    place(c);
    load_k();
    load_v();
    if (c + kPagedWaves < t.c_end)
      find(c + kPagedWaves);
  }
  for (; c < t.c_end; c += kPagedWaves) {
    const bool more = c + kPagedWaves < t.c_end;
    const bool own = c >= t.lead;
    const int key0 = (own ? c - t.lead : c) * kBlockKeys;
    const uint32_t live = there;
    if (pad_k) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        if (32 * ks + 8 * lg >= p.dqk)
          kf[0][ks] = kf[1][ks] = i32x4{0, 0, 0, 0};
    }
    f32x4 s[RF][2];
#pragma unroll
    for (int r = 0; r < RF; ++r)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        s[r][f] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          s[r][f] = Mfma16<f16>::mma(kf[f][ks], qf[r][ks], s[r][f]);
        s[r][f] *= scale;
      }
    if (live != 0xffffffffu || (own && key0 + kBlockKeys > all_own)) {
#pragma unroll
      for (int r = 0; r < RF; ++r) {
        const int end = own ? limit[r] : t.prefix;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = 16 * (e >> 2) + 4 * lg + (e & 3);
          if (key0 + key >= end || !(live >> key & 1))
            s[r][e >> 2][e & 3] = kNegInf;
        }
      }
    }
    if (more) {
      place(c + kPagedWaves);
      load_k();
      if (c + 2 * kPagedWaves < t.c_end)
        find(c + 2 * kPagedWaves);
    }

    float top[RF];
    bool move = false;
#pragma unroll
    for (int r = 0; r < RF; ++r) {
      float x = s[r][0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e)
        x = fmaxf(x, s[r][e >> 2][e & 3]);
      top[r] = x;
      move |= x > m_ref[r];
    }
    if (__any(move)) {
#pragma unroll
      for (int r = 0; r < RF; ++r) {
        const float x = fmaxf(m_ref[r], across_groups_max(top[r]));
        const float keep =
            x == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m_ref[r] - x);
        m_ref[r] = x;
        l_sum[r] *= keep;
#pragma unroll
        for (int d = 0; d < DB; ++d)
          o[r][d] *= keep;
      }
    }
    // The weights are rounded to f16 for the matrix instruction, by at most
    // 2^-11 of each and, the largest being 1, 2^-25 of the sum's least; the
    // sum is of the rounded ones.
    i32x4 pf[RF];
#pragma unroll
    for (int r = 0; r < RF; ++r) {
      const float ref = m_ref[r] == kNegInf ? 0.0f : m_ref[r];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x0 = s[r][e >> 1][2 * (e & 1)];
        const float x1 = s[r][e >> 1][2 * (e & 1) + 1];
        const f16x2 p2 = {(f16)__builtin_amdgcn_exp2f(x0 - ref),
                          (f16)__builtin_amdgcn_exp2f(x1 - ref)};
        l_sum[r] = __builtin_amdgcn_fdot2(p2, ones, l_sum[r], false);
        pf[r][e] = __builtin_bit_cast(int, p2);
      }
    }

    // V through this wave's LDS tile; keys that are not there are zeros.
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const int k = i * VROWS + vrow;
      if (!(live >> k & 1))
        vf[i] = i32x4{0, 0, 0, 0};
      *(i32x4 *)(vs + k * (DP * 2) + ((vch ^ v_swizzle<NCH>(k)) << 4)) = vf[i];
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
          (((byte >> 4) ^ v_swizzle<NCH>(k)) << 4) + (byte & 15);
      const i32x2 lo = __builtin_bit_cast(
          i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((IHP_LDS s16x4 *)at));
      const i32x2 hi = __builtin_bit_cast(
          i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                     (IHP_LDS s16x4 *)(at + 16 * (DP * 2))));
      const i32x4 v = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
      for (int r = 0; r < RF; ++r)
        o[r][d] = Mfma16<f16>::mma(v, pf[r], o[r][d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // Merge the waves: a common max per row, O scaled to it. A row whose
  // scores are all NaN has m -inf and l NaN, which the sums keep.
#pragma unroll
  for (int r = 0; r < RF; ++r) {
    const float l = across_groups_sum(l_sum[r]);
    if (lg == 0) {
      wave_m[wave][r * 16 + l15] = m_ref[r];
      wave_l[wave][r * 16 + l15] = l;
    }
  }
  __syncthreads();
  // Thread (q, dq) of the merge: row q of a fragment, DP / 16 columns from dq.
  constexpr int CPT = DP / 16;
  const int q = tid >> 4, dq = (tid & 15) * CPT;
#pragma unroll
  for (int r = 0; r < RF; ++r) {
    float *om = (float *)smem;
    {
      float top = kNegInf;
#pragma unroll
      for (int w = 0; w < kPagedWaves; ++w)
        top = fmaxf(top, wave_m[w][r * 16 + l15]);
      const float f =
          m_ref[r] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m_ref[r] - top);
#pragma unroll
      for (int d = 0; d < DB; ++d)
        *(f32x4 *)(om + (wave * 16 + l15) * OPITCH + 16 * d + 4 * lg) =
            o[r][d] * f;
    }
    __syncthreads();
    float top = kNegInf, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w)
      top = fmaxf(top, wave_m[w][r * 16 + q]);
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w)
      sum += wave_l[w][r * 16 + q] *
             (wave_m[w][r * 16 + q] == kNegInf
                  ? 0.0f
                  : __builtin_amdgcn_exp2f(wave_m[w][r * 16 + q] - top));
    float acc[CPT];
#pragma unroll
    for (int e = 0; e < CPT; ++e) {
      acc[e] = 0.0f;
#pragma unroll
      for (int w = 0; w < kPagedWaves; ++w)
        acc[e] += om[(w * 16 + q) * OPITCH + dq + e];
    }
    __syncthreads();  // before the next fragment's rows
    const int row = t.r0 + r * 16 + q;
    if (row >= t.r_end)
      continue;
    if (!p.partials) {
      const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
      f16 *dst = p.o + (int64_t)(row / p.group) * p.o_row +
                 (int64_t)(t.kv_head * p.group + row % p.group) * p.o_head + dq;
#pragma unroll
      for (int e = 0; e < CPT; e += 4)
        if (dq + e < p.dv)  // dv is a multiple of 8
          *(f16x4 *)(dst + e) =
              f16x4{(f16)(acc[e] * inv), (f16)(acc[e + 1] * inv),
                    (f16)(acc[e + 2] * inv), (f16)(acc[e + 3] * inv)};
    } else {
      const int64_t at =
          ((int64_t)t.part * p.kv_heads + t.kv_head) * p.packed + row;
      float *dst = p.partials + at * DP + dq;
#pragma unroll
      for (int e = 0; e < CPT; e += 4)
        *(f32x4 *)(dst + e) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
      if (dq == 0) {
        p.part_ml[2 * at] = top;
        p.part_ml[2 * at + 1] = sum;
      }
    }
  }
}

// Grid: the prefix's items (tile, KV head, split), then the requests' own.
template <int DP, int RP, int RO>
__global__ __launch_bounds__(kPagedThreads, DP >= 256 ? 1 : 2) void
attention_paged_kernel(PagedAttention p) {
  constexpr int VBYTES = kBlockKeys * DP * 2;
  constexpr int MERGE = kPagedWaves * 16 * (DP + 4) * 4;
  constexpr int SMEM = kPagedWaves * VBYTES > MERGE ? kPagedWaves * VBYTES : MERGE;
  __shared__ __attribute__((aligned(1024))) char smem[SMEM];
  __shared__ float wave_m[kPagedWaves][32], wave_l[kPagedWaves][32];
  const int prefix_items = p.prefix_tiles * p.kv_heads * p.prefix_splits;
  PagedTile t;
  t.prefix = p.prefix;
  const int prefix_blocks = (p.prefix + kBlockKeys - 1) / kBlockKeys;
  if ((int)blockIdx.x < prefix_items) {
    // Consecutive tiles of one (head, split) read the same keys: one XCD's.
    int item, unused;
    xcd_tile_order((int)blockIdx.x, prefix_items, prefix_items, 1, 1, &item,
                   &unused);
    const int tile = item % p.prefix_tiles, rest = item / p.prefix_tiles;
    t.part = rest % p.prefix_splits;
    t.kv_head = rest / p.prefix_splits;
    t.r0 = tile * (RP * 16);
    t.r_end = row_start(p, p.batch) * p.group;
    if (t.r0 >= t.r_end)
      return;
    t.lead = prefix_blocks;
    t.table = nullptr;
    t.own_end = t.base = t.first = 0;
    const int per = (prefix_blocks + p.prefix_splits - 1) / p.prefix_splits;
    t.c_begin = t.part * per;
    t.c_end = t.c_begin + per < prefix_blocks ? t.c_begin + per : prefix_blocks;
    paged_tile<DP, RP>(p, t, smem, wave_m, wave_l);
    return;
  }
  constexpr int RM = RO * 16;
  const int own_items = (int)gridDim.x - prefix_items;
  int item, unused;
  xcd_tile_order((int)blockIdx.x - prefix_items, own_items, own_items, 1, 1,
                 &item, &unused);
  const int tile = item % p.own_tiles, rest = item / p.own_tiles;
  const int split = rest % p.own_splits;
  t.kv_head = rest / p.own_splits;
  const int b = __builtin_amdgcn_readfirstlane(request_of<RM>(p, tile));
  const int begin = row_start(p, b), end = row_start(p, b + 1);
  const int64_t r0 = (int64_t)begin * p.group +
                     (int64_t)(tile - ((int64_t)begin * p.group / RM + b)) * RM;
  if (r0 < (int64_t)begin * p.group || r0 >= (int64_t)end * p.group)
    return;
  t.r0 = (int)r0;
  t.r_end = end * p.group;
  const int length = p.lengths[b];
  t.own_end = length < 0 ? 0 : length < p.capacity ? length : p.capacity;
  t.base = (length < 0 ? 0 : length) - (end - begin);
  t.first = begin;
  t.table = p.table + (int64_t)b * p.table_stride;
  // Blocks up to the last key that the tile's last row sees.
  const int r_last = t.r0 + RM < t.r_end ? t.r0 + RM - 1 : t.r_end - 1;
  int seen = t.base + r_last / p.group - begin + 1;
  seen = seen < 0 ? 0 : seen > t.own_end ? t.own_end : seen;
  t.lead = p.prefix_splits ? 0 : prefix_blocks;
  const int blocks = t.lead + (seen + kBlockKeys - 1) / kBlockKeys;
  int per = (blocks + p.own_splits - 1) / p.own_splits;
  per = per < kPagedSplitBlocks ? kPagedSplitBlocks : per;
  t.part = p.prefix_splits + split;
  t.c_begin = split * per < blocks ? split * per : blocks;
  t.c_end = blocks - t.c_begin < per ? blocks : t.c_begin + per;
  paged_tile<DP, RO>(p, t, smem, wave_m, wave_l);
}

// Joins the parts of every row: DP / 4 threads a row, 4 columns each.
template <int DP>
__global__ __launch_bounds__(kPagedThreads) void attention_paged_join_kernel(
    PagedAttention p) {
  constexpr int TPR = DP / 4;
  const int64_t at = (int64_t)blockIdx.x * (kPagedThreads / TPR) +
                     threadIdx.x / TPR;
  const int dq = 4 * ((int)threadIdx.x % TPR);
  const int kv_head = (int)(at / p.packed), row = (int)(at % p.packed);
  if (kv_head >= p.kv_heads || row >= row_start(p, p.batch) * p.group ||
      dq >= p.dv)
    return;
  const int parts = p.prefix_splits + p.own_splits;
  const int64_t step = (int64_t)p.kv_heads * p.packed;
  float top = kNegInf, sum = 0.0f;
  f32x4 acc = {0, 0, 0, 0};
  // 4 parts' loads in flight; a part past the last repeats it with weight 0
  for (int s0 = 0; s0 < parts; s0 += 4) {
    float m[4], l[4];
    f32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = at + (s0 + u < parts ? s0 + u : parts - 1) * step;
      m[u] = p.part_ml[2 * i];
      l[u] = p.part_ml[2 * i + 1];
      v[u] = *(const f32x4 *)(p.partials + i * DP + dq);
    }
    float x = top;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      x = fmaxf(x, m[u]);
    const float keep = top == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(top - x);
    top = x;
    sum *= keep;
    acc *= keep;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + u < parts) {
        const float f =
            m[u] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m[u] - x);
        sum += f * l[u];
        acc += f * v[u];
      }
  }
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  f16 *dst = p.o + (int64_t)(row / p.group) * p.o_row +
             (int64_t)(kv_head * p.group + row % p.group) * p.o_head + dq;
  *(f16x4 *)dst = f16x4{(f16)(acc[0] * inv), (f16)(acc[1] * inv),
                          (f16)(acc[2] * inv), (f16)(acc[3] * inv)};
}

// ----------------------------------------------------------------------------
// Host side.
// ----------------------------------------------------------------------------

namespace {

struct PagedKernel {
  const char *name;
  int dp, rp, ro;
  const void *fn;
};
#define IHP_PAGED(DP, RP, RO)                                                  \
  {"attention_paged_d" #DP "_r" #RP "_r" #RO, DP, RP, RO,                      \
   (const void *)&attention_paged_kernel<DP, RP, RO>}
const PagedKernel kPagedKernels[] = {
    IHP_PAGED(64, 2, 1),  IHP_PAGED(64, 2, 2),  IHP_PAGED(128, 2, 1),
    IHP_PAGED(128, 2, 2), IHP_PAGED(256, 1, 1),
};
constexpr int kPagedKernelCount =
    sizeof(kPagedKernels) / sizeof(kPagedKernels[0]);
const PagedKernel kJoinKernels[] = {
    {"attention_paged_join_d64", 64, 0, 0,
     (const void *)&attention_paged_join_kernel<64>},
    {"attention_paged_join_d128", 128, 0, 0,
     (const void *)&attention_paged_join_kernel<128>},
    {"attention_paged_join_d256", 256, 0, 0,
     (const void *)&attention_paged_join_kernel<256>},
};

}  // namespace

PagedPlan plan_attention_paged(int64_t rows, int64_t batch, int64_t kv_heads,
                               int64_t group, int64_t prefix, int64_t capacity,
                               int64_t head_dim, int64_t head_dim_v,
                               size_t workspace_limit) {
  PagedPlan p = {};
  const int64_t d = head_dim > head_dim_v ? head_dim : head_dim_v;
  p.dp = d <= 64 ? 64 : d <= 128 ? 128 : 256;
  const int64_t packed = rows * group;
  p.rp = p.dp < 256 ? 2 : 1;
  p.ro = p.dp < 256 && packed > 16 * batch ? 2 : 1;
  p.own_tiles = packed / (16 * p.ro) + batch;
  const int64_t part_bytes = kv_heads * packed * (p.dp + 2) * 4;
  const int64_t most_parts =
      workspace_limit <= kWorkspaceCounterBytes
          ? 0
          : (int64_t)((workspace_limit - kWorkspaceCounterBytes) /
                      (size_t)part_bytes);
  auto clamp = [](int64_t v, int64_t lo, int64_t hi) {
    return v < lo ? lo : v > hi ? hi : v;
  };
  const int64_t prefix_blocks = (prefix + kBlockKeys - 1) / kBlockKeys;
  const int64_t own_blocks = (capacity + kBlockKeys - 1) / kBlockKeys;
  // Requests whose rows fill tiles walk the prefix themselves.
  const bool shared = prefix > 0 && packed < 32 * batch && most_parts >= 2;
  int64_t own_keys = own_blocks + (shared ? 0 : prefix_blocks);
  p.own_splits = clamp(kPagedTargetWgs / (p.own_tiles * kv_heads), 1, 16);
  p.own_splits =
      clamp(p.own_splits, 1, (own_keys + kPagedSplitBlocks - 1) / kPagedSplitBlocks);
  if (shared) {
    p.prefix_tiles = (packed + 16 * p.rp - 1) / (16 * p.rp);
    p.prefix_splits =
        clamp(kPagedTargetWgs / (p.prefix_tiles * kv_heads), 1, 32);
    p.prefix_splits =
        clamp(p.prefix_splits, 1,
              (prefix_blocks + kPagedSplitBlocks - 1) / kPagedSplitBlocks);
    if (p.prefix_splits + p.own_splits > most_parts) {
      // as many parts as fit, the prefix's first
      p.own_splits = clamp(p.own_splits, 1, most_parts / 2);
      p.prefix_splits = clamp(p.prefix_splits, 1, most_parts - p.own_splits);
    }
  } else if (p.own_splits > 1) {
    p.own_splits = clamp(p.own_splits, 1, most_parts < 1 ? 1 : most_parts);
  }
  if (p.own_splits < 1)
    p.own_splits = 1;
  const int64_t parts = p.prefix_splits + p.own_splits;
  p.workspace =
      parts > 1 ? (int64_t)kWorkspaceCounterBytes + parts * part_bytes : 0;
  p.items = (p.prefix_tiles * p.prefix_splits + p.own_tiles * p.own_splits) *
            kv_heads;
  return p;
}

hipError_t launch_attention_paged(const PagedAttention &attention,
                                  const PagedPlan &plan, void *workspace,
                                  void *stream) {
  PagedAttention a = attention;
  a.prefix_tiles = (int)plan.prefix_tiles;
  a.prefix_splits = (int)plan.prefix_splits;
  a.own_tiles = (int)plan.own_tiles;
  a.own_splits = (int)plan.own_splits;
  const int64_t parts = plan.prefix_splits + plan.own_splits;
  const int64_t all = (int64_t)a.kv_heads * a.packed;
  a.partials = nullptr;
  a.part_ml = nullptr;
  if (parts > 1) {
    a.partials = (float *)((char *)workspace + kWorkspaceCounterBytes);
    a.part_ml = a.partials + parts * all * plan.dp;
  }
  const void *kernel = nullptr;
  for (const PagedKernel &k : kPagedKernels)
    if (k.dp == plan.dp && k.rp == plan.rp && k.ro == plan.ro)
      kernel = k.fn;
  if (!kernel)
    return hipErrorInvalidValue;
  void *args[] = {&a};
  hipError_t e = hipLaunchKernel(kernel, dim3((unsigned)plan.items),
                                 dim3(kPagedThreads), args, 0,
                                 (hipStream_t)stream);
  if (e != hipSuccess || parts == 1)
    return e;
  for (const PagedKernel &k : kJoinKernels)
    if (k.dp == plan.dp)
      kernel = k.fn;
  const int per = kPagedThreads / (plan.dp / 4);
  return hipLaunchKernel(kernel, dim3((unsigned)((all + per - 1) / per)),
                         dim3(kPagedThreads), args, 0, (hipStream_t)stream);
}

const KernelEntry *attention_paged_kernels(int *count) {
  constexpr int kJoins = sizeof(kJoinKernels) / sizeof(kJoinKernels[0]);
  static KernelEntry all[kPagedKernelCount + kJoins];
  static const bool filled = [] {
    for (int i = 0; i < kPagedKernelCount; ++i)
      all[i] = {kPagedKernels[i].name, kPagedKernels[i].fn, kPagedThreads, 0};
    for (int i = 0; i < kJoins; ++i)
      all[kPagedKernelCount + i] = {kJoinKernels[i].name, kJoinKernels[i].fn,
                                    kPagedThreads, 0};
    return true;
  }();
  (void)filled;
  *count = kPagedKernelCount + kJoins;
  return all;
}

}  // namespace ihp
