// Decode attention over quantised caches, and the entry points of the decode kernels of palu_step.h.
#include "palu_step.h"

namespace {

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int step_any(const StepArgs& a, int layout, const char* who, hipStream_t s) {
  if (layout == PALU_LAYOUT_MX8) return step_run<PALU_LAYOUT_MX8>(a, who, s);
  if (layout == PALU_LAYOUT_MX4) return step_run<PALU_LAYOUT_MX4>(a, who, s);
  return palu::step_bf16(a, layout, who, s);
}

// Everything but the prefixes and the workspace. `positions`: of a page (of a row without a page table).
int step_setup(StepArgs& a, const void* q, const void* k, const void* v, const int32_t* cur, void* out, float scale, int batch,
               int n_q, int n_kv, int positions, const int32_t* table, int pt_stride, int n_pages, int page_shift, int dv,
               int out_dtype, int layout, const char* who) {
  if (!q || !k || !v || !cur || !out) return fail(PALU_EINVAL, "%s: a required tensor pointer is null", who);
  if (batch <= 0 || n_q <= 0 || n_kv <= 0 || positions <= 0)
    return fail(PALU_EINVAL, "%s: batch, head counts and positions must be positive", who);
  if (n_q % n_kv != 0 || n_q / n_kv > 16)
    return fail(PALU_EINVAL, "KV head count %d must divide the %d query heads with at most 16 query heads per KV head", n_kv, n_q);
  if (out_dtype != PALU_DTYPE_F32 && out_dtype != PALU_DTYPE_BF16) return fail(PALU_EINVAL, "output dtype must be fp32 or bf16");
  const bool mx = layout == PALU_LAYOUT_MX8 || layout == PALU_LAYOUT_MX4;
  if (!mx && layout != PALU_LAYOUT_ROWS && layout != PALU_LAYOUT_TILED)
    return fail(PALU_EINVAL, "%s: cache layout must be PALU_LAYOUT_ROWS, _TILED, _MX8 or _MX4, got %d", who, layout);
  const int step = mx ? 32 : 16;
  if (dv < step || dv > HD || dv % step)
    return fail(PALU_EUNSUPPORTED, "%s: head_dim_v %d (multiples of %d up to %d)", who, dv, step, HD);
  if (positions % 32) return fail(PALU_EINVAL, "%s: a cache holds whole 32-position blocks, got %d positions", who, positions);
  const long long capacity = table ? (long long)pt_stride * positions : positions;
  if ((long long)batch * n_kv > 65535) return fail(PALU_EUNSUPPORTED, "batch * n_kv = %lld exceeds the grid limit", (long long)batch * n_kv);
  if (capacity > 65536) return fail(PALU_EUNSUPPORTED, "%s: %lld positions; this build covers 65536", who, capacity);
  if (!al16(q) || !al16(k) || !al16(v) || !al16(out)) return fail(PALU_EINVAL, "%s: 16-byte alignment required", who);
  memset(&a, 0, sizeof(a));
  const bool fp8 = layout == PALU_LAYOUT_MX8;
  a.q = static_cast<const __bf16*>(q);
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.k_blk = mx ? mx_block(fp8, HD) : 64 * HD;
  a.v_blk = mx ? mx_block(fp8, dv) : 64 * dv;
  a.k_head = (long long)(positions / 32) * a.k_blk;
  a.v_head = (long long)(positions / 32) * a.v_blk;
  a.k_page = a.k_head * n_kv;
  a.v_page = a.v_head * n_kv;
  a.cur = cur;
  a.table = table;
  a.pt_stride = pt_stride;
  a.n_pages = n_pages;
  a.page_shift = page_shift;
  a.capacity = (int)capacity;
  a.B = batch;
  a.n_q = n_q;
  a.n_kv = n_kv;
  a.rep = n_q / n_kv;
  a.dv = dv;
  a.qscale = scale * 1.4426950408889634f;
  a.out = out;
  a.f32_out = out_dtype == PALU_DTYPE_F32;
  return PALU_OK;
}

int step_workspace(StepArgs& a, void* workspace, size_t bytes, size_t need, const char* query, const char* who) {
  if (!workspace || bytes < need || !al16(workspace))
    return fail(PALU_EINVAL, "%s: a 16-byte aligned workspace of %zu bytes needed (%s), got %zu", who, need, query,
                workspace ? bytes : 0);
  const long long slots = step_slots(a.B, a.n_kv);
  a.part = static_cast<float*>(workspace);
  a.flags = reinterpret_cast<unsigned long long*>(a.part + slots * a.rep * (a.dv + 2));
  a.epoch = next_epoch();
  return PALU_OK;
}

bool step_dims(int batch, int n_q, int n_kv, int dv) {
  return batch > 0 && n_q > 0 && n_kv > 0 && dv > 0 && n_q % n_kv == 0 && n_q / n_kv <= 16 && dv <= HD && dv % 16 == 0 &&
         (long long)batch * n_kv <= 65535;
}
size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

namespace palu {

int mx_flash_decode(const void* q, const void* k, const void* v, const int32_t* cur_pos, void* out, float scale, int batch,
                    int n_q, int n_kv, int positions, const int32_t* page_table, int pt_stride, int n_pages, int page_shift,
                    int head_dim_v, int out_dtype, int layout, void* workspace, size_t workspace_bytes, const char* who,
                    hipStream_t stream) {
  StepArgs a;
  if (int rc = step_setup(a, q, k, v, cur_pos, out, scale, batch, n_q, n_kv, positions, page_table, pt_stride, n_pages, page_shift,
                          head_dim_v, out_dtype, layout, who))
    return rc;
  if (int rc = step_workspace(a, workspace, workspace_bytes, step_bytes(batch, n_kv, a.rep, head_dim_v),
                              "palu_mx_decode_workspace_bytes", who))
    return rc;
  return step_any(a, layout, who, stream);
}

}  // namespace palu

extern "C" size_t palu_mx_decode_workspace_bytes(int batch, int n_q, int n_kv, int head_dim_v) {
  return step_dims(batch, n_q, n_kv, head_dim_v) ? step_bytes(batch, n_kv, n_q / n_kv, head_dim_v) : 0;
}

extern "C" size_t palu_flash_decode_shared_workspace_bytes(int batch, int n_groups, int n_q, int n_kv, int head_dim_v) {
  if (!step_dims(batch, n_q, n_kv, head_dim_v) || n_groups <= 0) return 0;
  return align16(step_bytes(batch, n_kv, n_q / n_kv, head_dim_v)) + pre_bytes(batch, n_groups, n_q / n_kv, n_kv, head_dim_v);
}

extern "C" int palu_flash_decode_shared(const void* q, const void* k_pages, const void* v_pages, const int32_t* cur_pos,
                                        const int32_t* page_table, const int32_t* cu_groups, const int32_t* shared_len, void* out,
                                        float scale, int batch, int n_groups, int n_q, int n_kv, int num_pages, int page_size,
                                        int max_pages_per_seq, int head_dim_v, int out_dtype, int cache_layout, void* workspace,
                                        size_t workspace_bytes, hipStream_t stream) {
  palu::g_err[0] = 0;
  const char* who = "palu_flash_decode_shared";
  int shift = 0;
  if (int rc = palu::check_pages(page_table, num_pages, page_size, max_pages_per_seq, &shift, who)) return rc;
  StepArgs a;
  if (int rc = step_setup(a, q, k_pages, v_pages, cur_pos, out, scale, batch, n_q, n_kv, page_size, page_table,
                          max_pages_per_seq, num_pages, shift, head_dim_v, out_dtype, cache_layout, who))
    return rc;
  if (!shared_len) return fail(PALU_EINVAL, "%s: a required tensor pointer is null", who);
  if (n_groups <= 0 || (!cu_groups && n_groups != 1))
    return fail(PALU_EINVAL, "%s: %d groups (one without cu_groups)", who, n_groups);
  if (batch > 4096 || n_groups > 4096) return fail(PALU_EUNSUPPORTED, "%s: %d rows in %d groups (at most 4096)", who, batch, n_groups);
  if (int rc = step_workspace(a, workspace, workspace_bytes, palu_flash_decode_shared_workspace_bytes(batch, n_groups, n_q, n_kv, head_dim_v),
                              "palu_flash_decode_shared_workspace_bytes", who))
    return rc;
  const int C = pre_tile(batch, n_groups, a.rep);
  a.cu = cu_groups;
  a.shared = shared_len;
  a.n_groups = n_groups;
  a.pre_cols = 16 * C;
  a.pre_slots = (int)pre_slots(batch, n_groups, a.rep, n_kv, C);
  a.pre = reinterpret_cast<float*>(static_cast<char*>(workspace) + align16(step_bytes(batch, n_kv, a.rep, head_dim_v)));
  // Where all that the tables can name is little, each row reads its prefix by itself, by its group's table: 64 MiB or less take less
  // than a second launch and its join (both launches, and one: three rows of fp8 behind 100 positions 14.2 us, 7.8, behind 8000
  // 19.1, 16.0; 64 rows of tiles behind 128 positions, 67 MB, 20.3, 12.9; 16 rows over 71 MB, the prefixes nearly all of it, 18.7,
  // 21.2; 30 rows of fp4 over 65 MB 19.2, 19.2). Those are tables as wide as their longest row. The host knows the width and not what
  // is shared: under a table for 32768 positions short prefixes take both launches (the three rows behind 100 positions 13.7 us, 7.6
  // under one of 128; 16 rows with 8 KV heads behind 700 17.1, 11.9).
  const long long most = (long long)batch * n_kv * (a.capacity / 32) * (a.k_blk + a.v_blk);
  if (most > (64LL << 20))
    a.rows = reinterpret_cast<RowPrefix*>(a.pre + (long long)a.pre_slots * a.pre_cols * (head_dim_v + 2));
  return step_any(a, cache_layout, who, stream);
}
