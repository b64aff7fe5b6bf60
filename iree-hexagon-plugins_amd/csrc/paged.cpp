// C-ABI entry points of the paged KV cache (include/iree_mi355x_kernels.h):
// host-side argument checks, plans and launches.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/iree_mi355x_kernels.h"
#include "kernels_internal.h"

namespace ihp {

static bool aligned_to(const void *p, size_t a) {
  return ((uintptr_t)p % a) == 0;
}

// The element strides of one cache tensor: each head's rows within 2^32 * 16
// bytes of its first one.
static int check_cache_strides(const char *who, const char *name,
                               const iree_mi355x_kv_cache_t &c,
                               const int64_t *st, int64_t dim) {
  for (int i = 0; i < 3; ++i) {
    if (st[i] < 0)
      return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: negative %s stride", who,
                  name);
    if (st[i] % 8 != 0)
      return fail(IREE_MI355X_MISALIGNED,
                  "%s: %s strides must be multiples of 8 elements", who, name);
  }
  if (c.page_size > 1 && st[2] < dim)
    return fail(IREE_MI355X_INVALID_ARGUMENT,
                "%s: %s token stride %lld overlaps its rows", who, name,
                (long long)st[2]);
  const __int128 span =
      (__int128)(c.pages > 0 ? c.pages - 1 : 0) * (st[0] / 8) +
      (__int128)(c.page_size - 1) * (st[2] / 8);
  if (span > (__int128)UINT32_MAX || st[0] / 8 > (int64_t)UINT32_MAX ||
      st[2] / 8 > (int64_t)UINT32_MAX)
    return fail(IREE_MI355X_UNSUPPORTED,
                "%s: a head's rows of %s span more than 64 GiB", who, name);
  return IREE_MI355X_OK;
}

static int check_cache(const char *who, const iree_mi355x_kv_cache_t &c) {
  if (c.pages < 0 || c.page_size < 0 || c.kv_heads < 0 || c.head_dim < 0 ||
      c.head_dim_v < 0)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: negative extent", who);
  if (c.page_size < 1)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: page size 0", who);
  if (c.head_dim < 8 || c.head_dim > 256 || c.head_dim % 8 != 0 ||
      c.head_dim_v < 8 || c.head_dim_v > 256 || c.head_dim_v % 8 != 0)
    return fail(IREE_MI355X_UNSUPPORTED,
                "%s: head dims %lld / %lld (multiples of 8 up to 256 "
                "supported)",
                who, (long long)c.head_dim, (long long)c.head_dim_v);
  // Slots are 32-bit.
  if (c.kv_heads > 65535 || c.pages >= kMaxExtent ||
      c.page_size >= kMaxExtent ||
      (c.pages > 0 && c.page_size > (kMaxExtent - 1) / c.pages))
    return fail(IREE_MI355X_UNSUPPORTED, "%s: cache too large", who);
  if (c.pages > 0 && (!c.k || !c.v))
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned_to(c.k, 16) || !aligned_to(c.v, 16))
    return fail(IREE_MI355X_MISALIGNED,
                "%s: the caches must be 16-byte aligned", who);
  int st = check_cache_strides(who, "k", c, c.k_strides, c.head_dim);
  return st ? st : check_cache_strides(who, "v", c, c.v_strides, c.head_dim_v);
}

// n / d = (n * magic >> 32) >> shift for n below 2^31, d > 1: with 2^(l-1) < d
// <= 2^l and magic = floor(2^(31+l) / d) + 1 (below 2^32), the product is over
// the true quotient by less than 2^-l, which does not reach the next multiple
// of 1 / d.
static void divider(int64_t d, uint32_t *magic, int *shift) {
  int l = 1;
  while (((int64_t)1 << l) < d)
    ++l;
  *magic = (uint32_t)((((uint64_t)1 << (31 + l)) / (uint64_t)(d > 1 ? d : 2)) +
                      1);
  *shift = l - 1;
}

// A call's extents, as far as its plan goes by them.
static bool plannable(const iree_mi355x_paged_attention_t &a) {
  const iree_mi355x_kv_cache_t &c = a.cache;
  return a.rows > 0 && a.batch > 0 && a.heads > 0 && c.kv_heads > 0 &&
         a.heads % c.kv_heads == 0 && a.heads <= 65535 &&
         c.head_dim >= 8 && c.head_dim <= 256 && c.head_dim_v >= 8 &&
         c.head_dim_v <= 256 && c.page_size > 0 &&
         c.page_size < kMaxExtent && a.table_width >= 0 &&
         a.prefix_length >= 0 && a.prefix_length < kMaxExtent / 2 &&
         a.batch < kMaxExtent / 2 &&
         a.rows < kMaxExtent / 2 / (a.heads / c.kv_heads);
}

static int64_t own_capacity(const iree_mi355x_paged_attention_t &a) {
  const int64_t most = kMaxExtent / 2 - 1;
  return a.table_width > most / a.cache.page_size
             ? most
             : a.table_width * a.cache.page_size;
}

static PagedPlan plan_of(const iree_mi355x_paged_attention_t &a,
                         size_t workspace_limit) {
  const iree_mi355x_kv_cache_t &c = a.cache;
  return plan_attention_paged(a.rows, a.batch, c.kv_heads,
                              a.heads / c.kv_heads, a.prefix_length,
                              own_capacity(a), c.head_dim, c.head_dim_v,
                              workspace_limit);
}

}  // namespace ihp

using namespace ihp;

extern "C" {

int iree_mi355x_page_tables(const iree_mi355x_page_tables_t *a, void *stream) {
  const char *who = "page_tables";
  if (!a)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: null arguments", who);
  if (a->batch < 0 || a->free_count < 0 || a->table_width < 0 ||
      a->table_stride < 0 || a->rows < 0)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: negative extent", who);
  if (a->page_size < 1)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: page size %lld", who,
                (long long)a->page_size);
  if (a->batch >= kMaxExtent || a->rows >= kMaxExtent ||
      a->page_size >= kMaxExtent || a->table_width >= kMaxExtent ||
      (a->table_stride > 0 && a->batch > INT64_MAX / 8 / a->table_stride))
    return fail(IREE_MI355X_UNSUPPORTED, "%s: problem too large", who);
  if (a->batch > 1 && a->table_stride < a->table_width)
    return fail(IREE_MI355X_INVALID_ARGUMENT,
                "%s: table pitch %lld overlaps its rows", who,
                (long long)a->table_stride);
  if (!a->row_starts || !a->needed || (a->rows > 0 && !a->slots) ||
      (a->batch > 0 && (!a->cached || !a->added || !a->lengths ||
                        (a->table_width > 0 && !a->block_table))) ||
      (a->free_count > 0 && !a->free_pages))
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: null pointer", who);
  const void *all[8] = {a->cached, a->added,  a->free_pages, a->block_table,
                        a->row_starts, a->lengths, a->slots, a->needed};
  for (const void *p : all)
    if (!aligned_to(p, 4))
      return fail(IREE_MI355X_MISALIGNED,
                  "%s: operands must be aligned to their element size", who);
  PageTables t = {};
  t.cached = a->cached;
  t.added = a->added;
  t.free_pages = a->free_pages;
  t.table = a->block_table;
  t.row_starts = a->row_starts;
  t.lengths = a->lengths;
  t.slots = a->slots;
  t.needed = a->needed;
  t.batch = a->batch;
  t.free_count = a->free_count;
  t.width = a->table_width;
  t.table_stride = a->table_stride;
  t.rows = a->rows;
  t.page_size = (int)a->page_size;
  return launch_status(launch_page_tables(t, stream), who);
}

int iree_mi355x_append_kv_f16(const iree_mi355x_kv_cache_t *cache,
                              const void *k, const void *v, int64_t rows,
                              const int64_t k_strides[2],
                              const int64_t v_strides[2],
                              const int32_t *slots, void *stream) {
  const char *who = "append_kv";
  if (!cache || !k_strides || !v_strides)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: null arguments", who);
  const iree_mi355x_kv_cache_t &c = *cache;
  int st = check_cache(who, c);
  if (st)
    return st;
  if (rows < 0)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: negative extent", who);
  for (int i = 0; i < 2; ++i)
    if (k_strides[i] < 0 || v_strides[i] < 0)
      return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: negative stride", who);
  if (rows >= kMaxExtent)
    return fail(IREE_MI355X_UNSUPPORTED, "%s: problem too large", who);
  if (rows == 0 || c.kv_heads == 0 || c.pages == 0)
    return ok();
  if (!k || !v || !slots)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: null pointer", who);
  for (int i = 0; i < 2; ++i)
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0)
      return fail(IREE_MI355X_MISALIGNED,
                  "%s: strides must be multiples of 8 elements", who);
  if (!aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(slots, 4))
    return fail(IREE_MI355X_MISALIGNED, "%s: k/v must be 16-byte aligned",
                who);
  AppendKv p = {};
  p.k = (const _Float16 *)k;
  p.v = (const _Float16 *)v;
  p.k_cache = (_Float16 *)c.k;
  p.v_cache = (_Float16 *)c.v;
  p.slots = slots;
  p.rows = rows;
  p.slot_count = c.pages * c.page_size;
  for (int i = 0; i < 2; ++i) {
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.kc[i] = c.k_strides[i];
    p.vc[i] = c.v_strides[i];
  }
  p.kv_heads = (int)c.kv_heads;
  p.chunks_k = (int)(c.head_dim / 8);
  p.chunks_v = (int)(c.head_dim_v / 8);
  p.page_size = (int)c.page_size;
  return launch_status(launch_append_kv(p, stream), who);
}

int iree_mi355x_shared_prefix_attention_f16(
    const iree_mi355x_paged_attention_t *a, void *workspace,
    size_t workspace_bytes, void *stream) {
  const char *who = "shared_prefix_attention";
  if (!a)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: null arguments", who);
  if (a->flags)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: unknown flag bits 0x%x",
                who, a->flags);
  const iree_mi355x_kv_cache_t &c = a->cache;
  int st = check_cache(who, c);
  if (st)
    return st;
  if (a->rows < 0 || a->heads < 0 || a->batch < 0 || a->table_width < 0 ||
      a->table_stride < 0 || a->prefix_length < 0)
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: negative extent", who);
  if (!std::isfinite(a->scale))
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: scale not finite", who);
  for (int i = 0; i < 2; ++i)
    if (a->q_strides[i] < 0 || a->o_strides[i] < 0)
      return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: negative stride", who);
  if (a->rows == 0 || a->heads == 0 || a->batch == 0)
    return ok();
  if (c.kv_heads == 0 || a->heads % c.kv_heads != 0)
    return fail(IREE_MI355X_INVALID_ARGUMENT,
                "%s: %lld query heads are not a multiple of %lld KV heads",
                who, (long long)a->heads, (long long)c.kv_heads);
  if (!plannable(*a) ||
      (a->table_stride > 0 && a->batch > INT64_MAX / 8 / a->table_stride))
    return fail(IREE_MI355X_UNSUPPORTED, "%s: problem too large", who);
  if (a->batch > 1 && a->table_stride < a->table_width)
    return fail(IREE_MI355X_INVALID_ARGUMENT,
                "%s: table pitch %lld overlaps its rows", who,
                (long long)a->table_stride);
  if (!a->q || !a->o || !a->row_starts || !a->lengths ||
      (a->table_width > 0 && !a->block_table) ||
      (a->prefix_length > 0 && !a->prefix_pages))
    return fail(IREE_MI355X_INVALID_ARGUMENT, "%s: null pointer", who);
  if ((a->heads > 1 && a->o_strides[1] < c.head_dim_v) ||
      (a->rows > 1 && a->o_strides[0] < c.head_dim_v))
    return fail(IREE_MI355X_INVALID_ARGUMENT,
                "%s: o strides %lld, %lld overlap its rows", who,
                (long long)a->o_strides[0], (long long)a->o_strides[1]);
  for (int i = 0; i < 2; ++i)
    if (a->q_strides[i] % 8 != 0 || a->o_strides[i] % 4 != 0)
      return fail(IREE_MI355X_MISALIGNED,
                  "%s: strides must be multiples of 8 elements (q), 4 (o)",
                  who);
  if (!aligned_to(a->q, 16) || !aligned_to(a->o, 8) ||
      !aligned_to(workspace, 16))
    return fail(IREE_MI355X_MISALIGNED,
                "%s: q and the workspace must be 16-byte aligned, o 8", who);
  if (!aligned_to(a->row_starts, 4) || !aligned_to(a->lengths, 4) ||
      !aligned_to(a->block_table, 4) || !aligned_to(a->prefix_pages, 4))
    return fail(IREE_MI355X_MISALIGNED,
                "%s: tables must be aligned to their element size", who);

  PagedAttention p = {};
  p.q = (const _Float16 *)a->q;
  p.o = (_Float16 *)a->o;
  p.k_cache = (const _Float16 *)c.k;
  p.v_cache = (const _Float16 *)c.v;
  p.row_starts = a->row_starts;
  p.lengths = a->lengths;
  p.table = a->block_table;
  p.prefix_pages = a->prefix_pages;
  p.q_row = a->q_strides[0];
  p.q_head = a->q_strides[1];
  p.o_row = a->o_strides[0];
  p.o_head = a->o_strides[1];
  p.k_head = c.k_strides[1];
  p.v_head = c.v_strides[1];
  p.table_stride = a->table_stride;
  p.k_page16 = (uint32_t)(c.k_strides[0] / 8);
  p.k_row16 = (uint32_t)(c.k_strides[2] / 8);
  p.v_page16 = (uint32_t)(c.v_strides[0] / 8);
  p.v_row16 = (uint32_t)(c.v_strides[2] / 8);
  divider(c.page_size, &p.page_magic, &p.page_shift);
  p.page_size = (int)c.page_size;
  p.pages = (int)c.pages;
  const int64_t small = (int64_t)1 << 24;
  auto reach = [&](const int64_t *st, int64_t dim) {  // bytes, head 0's rows
    return ((c.pages > 0 ? c.pages - 1 : 0) * st[0] +
            (c.page_size - 1) * st[2] + dim) * 2;
  };
  p.near = c.pages <= small && c.page_size <= small &&
           p.k_page16 < small && p.k_row16 < small && p.v_page16 < small &&
           p.v_row16 < small && reach(c.k_strides, 256) < UINT32_MAX &&
           reach(c.v_strides, 256) < UINT32_MAX;
  p.batch = (int)a->batch;
  p.rows = (int)a->rows;
  p.kv_heads = (int)c.kv_heads;
  p.group = (int)(a->heads / c.kv_heads);
  p.packed = a->rows * p.group;
  divider(p.group, &p.group_magic, &p.group_shift);
  p.narrow_tokens = 16 / p.group;
  p.wide_tokens = 128 / p.group;
  p.dqk = (int)c.head_dim;
  p.dv = (int)c.head_dim_v;
  // A cache without pages has no keys.
  p.prefix = c.pages > 0 ? (int)a->prefix_length : 0;
  p.capacity = c.pages > 0 ? (int)own_capacity(*a) : 0;
  p.scale = a->scale;
  iree_mi355x_paged_attention_t b = *a;
  if (c.pages == 0)
    b.prefix_length = b.table_width = 0;
  const PagedPlan plan = plan_of(b, workspace ? workspace_bytes : 0);
  // A launch has fewer than 2^32 threads.
  const int64_t most = (int64_t)1 << 24;
  if (plan.ways * c.kv_heads >= most ||
      (plan.workspace && p.packed * p.kv_heads / (1024 / plan.dp) >= most - 1))
    return fail(IREE_MI355X_UNSUPPORTED, "%s: problem too large", who);
  return launch_status(launch_attention_paged(p, plan, workspace, stream),
                       who);
}

size_t iree_mi355x_shared_prefix_attention_workspace_bytes(
    const iree_mi355x_paged_attention_t *a) {
  if (!a || !plannable(*a))
    return 0;
  return (size_t)plan_of(*a, (size_t)-1).workspace;
}

}  // extern "C"
