// The paged KV cache's tables and the rows appended to it.
//
// page_tables_kernel: from the tokens that each request has in its pages and
// those it adds, the packed rows' starts, the lengths after the step, the
// pages taken from the free list into the block table, and the slot (page *
// page size + place) of every new row. With up(x) = ceil(x / page size):
//   row_starts[b] = sum_{i<b} added[i]
//   take[b] = up(cached[b] + added[b]) - up(cached[b]), as far as the
//     table's row goes
//   block_table[b][up(cached[b]) + j] = free[sum_{i<b} take[i] + j]
//   slots[row_starts[b] + i] = place of token cached[b] + i
// One launch: every workgroup scans all requests by itself, 512 at a time
// (both prefix sums in one pass over the waves), and writes the rows and
// table entries that fall to it, finding their request by bisection in LDS.
// Nothing is exchanged between workgroups, so there is no second launch and
// no counter. Bound by its chain of loads and barriers: 3.7 us for one
// request, 4.8 for 256, 7.6 for 48 with 55832 new rows.
//
// append_kv_kernel: rows of K and V into the pages that the slots name,
// 16 bytes a lane. A row whose slot lies outside the cache is skipped. Bound
// by memory: 8191 rows of 8 heads (67 MB) in 11.5 us, 5.8 TB/s; 64 rows 3.4.
//
// tree_masks_kernel: which of its request's new rows each one of a tree sees,
// from the rows' parents. A wave takes a request, 64 rows at a time: with p(i)
// the parent of row i,
//   seen(i) = {i} + seen(p(i)),  depth(i) = 1 + depth(p(i))
// and within the 64 rows the ancestors of all come from six doublings,
//   seen_k+1(i) = seen_k(i) + seen_k(p^(2^k)(i))
// as a 64-bit set a lane. The first ancestor before the 64 rows is the parent
// of the topmost one among them, and its mask and depth are known by then: in
// LDS, as far as it holds a request's (4096 words), else in the output. Bound by
// the chain of 64s in the longest request: 32 trees of 9 to 63 nodes 2.9 us, 48 of
// up to 250 beside a chain of 500, 8 words, 9 to 10 (with the masks read back from
// memory 14 to 16). A chain of 2048 takes 29 us, of 8192 112 (2 words, a call among
// others).
#include "device_common.h"
#include "kernels_internal.h"

namespace ihp {

namespace {

constexpr int kTableThreads = 512;
constexpr int kTableWaves = kTableThreads / 64;
constexpr int kAppendThreads = 256;
constexpr int kMaskThreads = 256;
constexpr int kMaskWaves = kMaskThreads / 64;
constexpr int kMaskWords = 4096;

__device__ __forceinline__ int32_t saturated(int64_t v) {
  return v > INT32_MAX ? INT32_MAX : (int32_t)v;
}

// The last i < n with start[i] <= x; start ascends from start[0] <= x.
__device__ __forceinline__ int bisect(const int64_t *start, int n, int64_t x) {
  int lo = 0;
  for (int step = kTableThreads / 2; step > 0; step >>= 1)
    if (lo + step < n && start[lo + step] <= x)
      lo += step;
  return lo;
}

}  // namespace

__global__ __launch_bounds__(kTableThreads) void page_tables_kernel(
    PageTables t) {
  __shared__ int64_t row_start[kTableThreads], page_start[kTableThreads];
  __shared__ uint32_t had[kTableThreads];
  __shared__ int64_t wave_rows[kTableWaves], wave_pages[kTableWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t page = (uint32_t)t.page_size;
  const int64_t stride = (int64_t)gridDim.x * kTableThreads;
  const int64_t mine = (int64_t)blockIdx.x * kTableThreads + tid;
  int64_t rows_before = 0, pages_before = 0;

  for (int64_t b0 = 0; b0 < t.batch; b0 += kTableThreads) {
    const int n =
        t.batch - b0 < kTableThreads ? (int)(t.batch - b0) : kTableThreads;
    uint32_t cached = 0, added = 0;
    if (tid < n) {
      const int32_t c = t.cached[b0 + tid], a = t.added[b0 + tid];
      cached = c > 0 ? (uint32_t)c : 0;
      added = a > 0 ? (uint32_t)a : 0;
    }
    const uint32_t length = cached + added;  // below 2^32
    const uint32_t width = (uint32_t)t.width;
    const uint32_t held = cached / page + (cached % page != 0);
    const uint32_t ends = length / page + (length % page != 0);
    const uint32_t take =
        (ends < width ? ends : width) - (held < width ? held : width);
    // Inclusive sums over the wave, then over the waves before it.
    int64_t rows = added, pages = take;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t r = __shfl_up(rows, d), p = __shfl_up(pages, d);
      if (lane >= d) {
        rows += r;
        pages += p;
      }
    }
    if (lane == 63) {
      wave_rows[wave] = rows;
      wave_pages[wave] = pages;
    }
    __syncthreads();
    int64_t rows_all = 0, pages_all = 0;
#pragma unroll
    for (int w = 0; w < kTableWaves; ++w) {
      if (w < wave) {
        rows += wave_rows[w];
        pages += wave_pages[w];
      }
      rows_all += wave_rows[w];
      pages_all += wave_pages[w];
    }
    rows += rows_before - added;  // this request's first row and page
    pages += pages_before - take;
    row_start[tid] = rows;
    page_start[tid] = pages;
    had[tid] = cached;
    if (tid < n && (b0 / kTableThreads) % gridDim.x == blockIdx.x) {
      t.row_starts[b0 + tid] = saturated(rows);
      t.lengths[b0 + tid] = saturated(length);
    }
    __syncthreads();

    // Pages taken by these requests.
    for (int64_t e = pages_before / stride * stride + mine;
         e < pages_before + pages_all; e += stride) {
      if (e < pages_before)
        continue;
      const int i = bisect(page_start, n, e);
      const uint32_t c = had[i];
      // below the width: none is taken past it
      const int64_t column =
          (int64_t)(c / page) + (c % page != 0) + (e - page_start[i]);
      t.table[(b0 + i) * t.table_stride + column] =
          e < t.free_count ? t.free_pages[e] : -1;
    }
    // Their rows' slots: a page taken by this call is read from the free
    // list, the request's last partly filled one from the table, which this
    // call leaves alone there.
    const int64_t rows_end = rows_before + rows_all < t.rows
                                 ? rows_before + rows_all
                                 : t.rows;
    for (int64_t r = rows_before / stride * stride + mine; r < rows_end;
         r += stride) {
      if (r < rows_before)
        continue;
      const int i = bisect(row_start, n, r);
      const uint32_t c = had[i];
      const uint32_t at = c + (uint32_t)(r - row_start[i]);
      const uint32_t column = at / page, had_pages = c / page + (c % page != 0);
      int64_t named = -1;
      if (column < t.width) {
        if (column < had_pages) {
          named = t.table[(b0 + i) * t.table_stride + column];
        } else {
          const int64_t e = page_start[i] + (column - had_pages);
          named = e < t.free_count ? t.free_pages[e] : -1;
        }
      }
      const int64_t slot = named * page + at % page;
      t.slots[r] = named < 0 || slot > INT32_MAX ? -1 : (int32_t)slot;
    }
    rows_before += rows_all;
    pages_before += pages_all;
    __syncthreads();  // before the next requests' sums
  }
  for (int64_t r = rows_before / stride * stride + mine; r < t.rows;
       r += stride)
    if (r >= rows_before)
      t.slots[r] = -1;
  if (blockIdx.x == 0 && tid == 0) {
    t.row_starts[t.batch] = saturated(rows_before);
    t.needed[0] = saturated(pages_before);
  }
}

__global__ __launch_bounds__(kAppendThreads) void append_kv_kernel(
    AppendKv a) {
  // A wave takes one row at a time, its lanes the row's 16-byte chunks: K's
  // heads, then V's.
  const int lane = threadIdx.x & 63;
  const int chunks_k = a.kv_heads * a.chunks_k, chunks_v = a.kv_heads * a.chunks_v;
  const int64_t waves = (int64_t)gridDim.x * (kAppendThreads / 64);
  for (int64_t row = (int64_t)blockIdx.x * (kAppendThreads / 64) +
                     (threadIdx.x >> 6);
       row < a.rows; row += waves) {
    const int32_t slot = a.slots[row];
    if (slot < 0 || slot >= a.slot_count)
      continue;
    const int64_t page = slot / a.page_size, place = slot % a.page_size;
    for (int c = lane; c < chunks_k; c += 64) {
      const int head = c / a.chunks_k, ch = c % a.chunks_k;
      *(i32x4 *)(a.k_cache + page * a.kc[0] + head * a.kc[1] + place * a.kc[2] +
                 8 * ch) =
          *(const i32x4 *)(a.k + row * a.ks[0] + head * a.ks[1] + 8 * ch);
    }
    for (int c = lane; c < chunks_v; c += 64) {
      const int head = c / a.chunks_v, ch = c % a.chunks_v;
      *(i32x4 *)(a.v_cache + page * a.vc[0] + head * a.vc[1] + place * a.vc[2] +
                 8 * ch) =
          *(const i32x4 *)(a.v + row * a.vs[0] + head * a.vs[1] + 8 * ch);
    }
  }
}

// Words that a row takes in LDS: its mask and its depth, an odd number.
__device__ __forceinline__ int mask_pitch(const TreeMasks &t) {
  return (t.words + 1) | 1;
}

// A request's rows. HELD: `held` has room for their masks and depths.
template <bool HELD>
__device__ __forceinline__ void tree_masks_of(const TreeMasks &t, int first,
                                              int end, int32_t *held) {
  const int lane = threadIdx.x & 63, pitch = mask_pitch(t);
  const bool fours =
      t.words % 4 == 0 && (uintptr_t)t.masks % 16 == 0;  // of words
  int next = first + lane < end ? t.parents[first + lane] : -1;
  for (int r0 = first; r0 < end; r0 += 64) {
    // node numbers within the request; a parent that is not an earlier one of
    // it is none
    const int i0 = r0 - first, i = i0 + lane;
    const bool real = r0 + lane < end;
    int parent = next;
    next = r0 + 64 + lane < end ? t.parents[r0 + 64 + lane] : -1;
    if (parent < 0 || parent >= i)
      parent = -1;
    uint64_t seen = 1ull << lane;
    int jump = parent - i0;
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      const int from = jump < 0 ? lane : jump;
      const uint64_t theirs =
          (uint64_t)(uint32_t)__shfl((int)(seen >> 32), from) << 32 |
          (uint32_t)__shfl((int)seen, from);
      const int further = __shfl(jump, from);
      if (jump >= 0) {
        seen |= theirs;
        jump = further;
      }
    }
    const int above = __shfl(parent, __builtin_ctzll(seen));
    // what this wave wrote of the rows before (LDS keeps a wave's order)
    if (HELD)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    else
      __threadfence_block();
    const int from = above < 0 ? 0 : above;
    const int64_t row = r0 + lane;
    const int32_t *theirs = HELD ? held + from * pitch
                                 : t.masks + (int64_t)(first + from) * t.words;
    int32_t *mine = HELD ? held + i * pitch : nullptr;
    int depth = HELD ? theirs[t.words] : t.depths[first + from];
    depth = (above < 0 ? -1 : depth) + __popcll(seen);
    if (real) {
      t.depths[row] = depth;
      if (HELD)
        mine[t.words] = depth;
    }
    for (int w0 = 0; w0 < t.words; w0 += 4) {
      i32x4 bits;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int word = theirs[w0 + j < t.words ? w0 + j : t.words - 1];
        // and bits 32 w .. of the nodes i0 .. i0 + 63
        const int shift = i0 - 32 * (w0 + j);
        bits[j] = (above < 0 ? 0 : word) | (shift == 0     ? (int)seen
                                            : shift == -32 ? (int)(seen >> 32)
                                                           : 0);
      }
      if (!real)
        continue;
      int32_t *out = t.masks + row * t.words + w0;
      if (fours)
        *(i32x4 *)out = bits;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w0 + j < t.words) {
          if (HELD)
            mine[w0 + j] = bits[j];
          if (!fours)
            out[j] = bits[j];
        }
    }
  }
}

__global__ __launch_bounds__(kMaskThreads) void tree_masks_kernel(
    TreeMasks t) {
  const int lane = threadIdx.x & 63;
  const int b = __builtin_amdgcn_readfirstlane(
      (int)(blockIdx.x * kMaskWaves + (threadIdx.x >> 6)));
  auto start = [&](int i) {  // within the rows that there are
    const int r = t.row_starts[i];
    return r < 0 ? 0 : r > t.rows ? t.rows : r;
  };
  if (b >= t.batch) {  // rows behind the last request
    const int64_t first = start(t.batch), end = t.rows;
    const int64_t step =
        ((int64_t)gridDim.x * kMaskWaves - t.batch) * 64;
    const int64_t mine = (int64_t)(b - t.batch) * 64 + lane;
    for (int64_t i = first * t.words + mine; i < end * t.words; i += step)
      t.masks[i] = 0;
    for (int64_t r = first + mine; r < end; r += step)
      t.depths[r] = 0;
    return;
  }
  __shared__ int32_t held_all[kMaskWaves][kMaskWords];
  const int first = start(b), end = start(b + 1);
  if ((int64_t)(end - first) * mask_pitch(t) <= kMaskWords)
    tree_masks_of<true>(t, first, end, held_all[threadIdx.x >> 6]);
  else
    tree_masks_of<false>(t, first, end, nullptr);
}

hipError_t launch_tree_masks(const TreeMasks &masks, void *stream) {
  TreeMasks t = masks;
  // Waves for the rows behind the last request, were it all: 16 words a lane.
  int64_t rest = ((int64_t)t.rows * t.words + 1023) / 1024;
  rest = rest > 64 ? 64 : rest;
  const int64_t wgs = (t.batch + rest + kMaskWaves - 1) / kMaskWaves;
  void *args[] = {&t};
  return hipLaunchKernel((const void *)&tree_masks_kernel,
                         dim3((unsigned)wgs), dim3(kMaskThreads), args, 0,
                         (hipStream_t)stream);
}

hipError_t launch_page_tables(const PageTables &tables, void *stream) {
  PageTables t = tables;
  const int64_t most = t.rows > t.batch ? t.rows : t.batch;
  // 4 rows a thread (55832 rows: 8.9 us a call, with 1 the same, 16 16.6).
  int64_t wgs = (most + kTableThreads * 4 - 1) / (kTableThreads * 4);
  wgs = wgs < 1 ? 1 : wgs > 256 ? 256 : wgs;
  void *args[] = {&t};
  return hipLaunchKernel((const void *)&page_tables_kernel,
                         dim3((unsigned)wgs), dim3(kTableThreads), args, 0,
                         (hipStream_t)stream);
}

hipError_t launch_append_kv(const AppendKv &append, void *stream) {
  AppendKv a = append;
  int64_t wgs = (a.rows + kAppendThreads / 64 - 1) / (kAppendThreads / 64);
  wgs = wgs > 2048 ? 2048 : wgs;  // 1024 and 8192: the same within 4 %
  void *args[] = {&a};
  return hipLaunchKernel((const void *)&append_kv_kernel, dim3((unsigned)wgs),
                         dim3(kAppendThreads), args, 0, (hipStream_t)stream);
}

const KernelEntry *paged_cache_kernels(int *count) {
  static const KernelEntry all[] = {
      {"page_tables", (const void *)&page_tables_kernel, kTableThreads, 0},
      {"append_kv", (const void *)&append_kv_kernel, kAppendThreads, 0},
      {"tree_masks", (const void *)&tree_masks_kernel, kMaskThreads, 0},
  };
  *count = (int)(sizeof(all) / sizeof(all[0]));
  return all;
}

}  // namespace ihp
