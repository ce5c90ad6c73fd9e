// extern "C" boundary of the paged cache and of beam selection: argument checks.  Declarations are in
// include/selective_attention_b200.h.
#include <mutex>

#include "sa_beam.cuh"
#include "sa_paged.cuh"
#include "sa_tc_host.cuh"

namespace sa {
namespace {

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int to_tables(const sa_page_tables* in, paged::Tables* t) {
  if (in == nullptr || in->struct_bytes != (int32_t)sizeof(sa_page_tables)) return SA_ERR_BAD_ARGUMENT;
  if (in->rows < 1 || in->max_pages < 1 || in->num_pages < 1 || in->heads < 1) return SA_ERR_BAD_ARGUMENT;
  int shift = 4;
  while (shift < 8 && (1 << shift) != in->page_size) ++shift;
  if ((1 << shift) != in->page_size || in->rows > paged::kMaxRows || in->heads > 256) return SA_ERR_UNSUPPORTED;
  // positions and slots are 32-bit numbers on the device
  if ((int64_t)in->max_pages * in->page_size > 0x7fffff00LL || (int64_t)in->num_pages * in->page_size > 0x7fffff00LL ||
      (int64_t)in->rows * in->max_pages > 0x7fffff00LL)
    return SA_ERR_TOO_LARGE;
  if (!in->block_tables || !in->lengths || !in->free_pages || !in->free_count || !in->page_refs) return SA_ERR_BAD_ARGUMENT;
  for (const void* p : {in->block_tables, in->lengths, in->free_pages, in->free_count, in->page_refs})
    if (!aligned(p, 4)) return SA_ERR_ALIGNMENT;
  *t = paged::Tables{in->rows, in->max_pages, in->num_pages, shift, in->heads, in->block_tables, in->lengths, in->free_pages, in->free_count,
                     in->page_refs};
  return SA_OK;
}

int to_attention(const sa_paged_attention* in, paged::Attention* a) {
  if (in == nullptr || in->struct_bytes != (int32_t)sizeof(sa_paged_attention)) return SA_ERR_BAD_ARGUMENT;
  paged::Tables t;
  const int st = to_tables(in->tables, &t);
  if (st != SA_OK) return st;
  if (in->groups < 1 || in->exempt < 1 || in->total < 1 || in->max_length < 1 || in->max_count < 1) return SA_ERR_BAD_ARGUMENT;
  if ((in->groups != 1 && in->groups != t.heads) || (in->head_dim != 64 && in->head_dim != 128)) return SA_ERR_UNSUPPORTED;
  if (in->max_length > (int64_t)t.max_pages << t.page_shift) return SA_ERR_BAD_ARGUMENT;
  *a = paged::Attention{};
  a->rows = t.rows; a->max_pages = t.max_pages; a->num_pages = t.num_pages; a->page_shift = t.page_shift;
  a->heads = t.heads; a->groups = in->groups; a->head_dim = in->head_dim; a->exempt = in->exempt;
  a->total = in->total; a->max_length = in->max_length; a->max_count = in->max_count < in->total ? in->max_count : in->total;
  a->block_tables = t.block_tables;
  a->sel_stride = (int64_t)t.max_pages << t.page_shift;
  const paged::StepLayout l = paged::step_layout(t.rows, in->total, t.heads);
  if ((int64_t)l.decode_items_max * t.heads > 0x7fffffffLL || (int64_t)l.tile_items_max * t.heads > 0x7fffffffLL ||
      (in->max_length + 127) / 128 / 8 > 65534)
    return SA_ERR_TOO_LARGE;
  return SA_OK;
}

}  // namespace
}  // namespace sa

using namespace sa;

extern "C" {

size_t sa_page_step_words(int rows, int total, int heads) {
  if (rows < 1 || rows > paged::kMaxRows || total < 0 || total > (1 << 30) || heads < 1 || heads > 256) return 0;
  return paged::step_layout(rows, total, heads).words;
}

int sa_page_append(const sa_page_tables* tables, const int32_t* counts, int total, int max_length, int max_count, int32_t* query_start,
                   int32_t* cached, int64_t* slots, int32_t* work, void* stream) {
  paged::Tables t;
  const int st = to_tables(tables, &t);
  if (st != SA_OK) return st;
  if (!counts || !query_start || !cached || !work || total < 0 || (total > 0 && !slots) || max_length < 1 || max_count < 1)
    return SA_ERR_BAD_ARGUMENT;
  if (total > (1 << 30)) return SA_ERR_TOO_LARGE;
  if (!aligned(work, 16) || !aligned(slots, 8)) return SA_ERR_ALIGNMENT;
  return paged::append(t, counts, total, max_length, max_count, query_start, cached, slots, work, static_cast<cudaStream_t>(stream));
}

size_t sa_page_reorder_words(int rows, int max_pages, int num_pages) {
  if (rows < 1 || rows > paged::kMaxRows || max_pages < 1 || num_pages < 1) return 0;
  return paged::reorder_work_words(rows, max_pages, num_pages);
}

int sa_page_reorder(const sa_page_tables* tables, const int32_t* parents, int32_t* copies, int32_t* work, void* stream) {
  paged::Tables t;
  const int st = to_tables(tables, &t);
  if (st != SA_OK) return st;
  if (!parents || !copies || !work) return SA_ERR_BAD_ARGUMENT;
  if (!aligned(work, 16) || !aligned(copies, 8)) return SA_ERR_ALIGNMENT;
  return paged::reorder(t, parents, copies, work, static_cast<cudaStream_t>(stream));
}

int sa_page_move(const sa_page_tables* tables, const int32_t* copies, const int32_t* work, int groups, int head_dim, void* k_pages,
                 void* v_pages, float* selected, void* stream) {
  paged::Tables t;
  const int st = to_tables(tables, &t);
  if (st != SA_OK) return st;
  if (!copies || !work || !k_pages || !v_pages || !selected || groups < 1 || head_dim < 1) return SA_ERR_BAD_ARGUMENT;
  if (head_dim % 8 != 0 || groups > 65535) return SA_ERR_UNSUPPORTED;
  if (!aligned(work, 16) || !aligned(copies, 8) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(selected, 16))
    return SA_ERR_ALIGNMENT;
  return paged::move_rows(t, copies, work, groups, head_dim, 2, (int64_t)t.max_pages << t.page_shift, k_pages, v_pages, selected,
                          static_cast<cudaStream_t>(stream));
}

size_t sa_paged_workspace_bytes(const sa_paged_attention* in) {
  paged::Attention a;
  return to_attention(in, &a) == SA_OK ? paged::attention_scratch(a).floats * 4 : 0;
}

int sa_paged_run(const sa_paged_attention* in) {
  paged::Attention a;
  int st = to_attention(in, &a);
  if (st != SA_OK) return st;
  if (!in->slots || !in->work || !in->q || !in->k || !in->v || !in->k_pages || !in->v_pages || !in->selected || !in->y || !in->workspace)
    return SA_ERR_BAD_ARGUMENT;
  for (const void* p : {in->q, in->k, in->v, (const void*)in->k_pages, (const void*)in->v_pages, (const void*)in->y, (const void*)in->work})
    if (!aligned(p, 16)) return SA_ERR_ALIGNMENT;
  if (!aligned(in->workspace, 256) || !aligned(in->selected, 4)) return SA_ERR_ALIGNMENT;
  for (const int64_t* s : {in->q_stride, in->k_stride, in->v_stride})
    if (s[0] % 8 != 0 || s[1] % 8 != 0 || s[0] <= 0 || s[1] <= 0) return SA_ERR_ALIGNMENT;
  if (in->workspace_bytes < paged::attention_scratch(a).floats * 4) return SA_ERR_WORKSPACE;
  if (tc::timeout_pending()) return SA_ERR_DEVICE_TIMEOUT;
  a.slots = in->slots; a.work = in->work;
  a.plan_tickets = in->plan_tickets != 0;
  a.k_pages = in->k_pages; a.v_pages = in->v_pages; a.selected = in->selected;
  a.q = in->q; a.k = in->k; a.v = in->v; a.y = in->y;
  for (int i = 0; i < 2; ++i) {
    a.q_stride[i] = in->q_stride[i];
    a.k_stride[i] = in->k_stride[i];
    a.v_stride[i] = in->v_stride[i];
  }
  a.workspace = static_cast<float*>(in->workspace);
  cudaStream_t s = static_cast<cudaStream_t>(in->stream);
  // A call's launches stand together in its stream: with another thread's between them, the few tokens of two calls could run at
  // once, and calls of one plan and stream share its tickets.
  static std::mutex launches;
  const std::lock_guard<std::mutex> guard(launches);
  // Rows of few tokens go through a kernel of their own, the others through the tile kernels; the step's bounds say where there can
  // be none of either.
  if (paged::few_only(a.total, a.max_count)) return paged::decode(a, false, s);
  bool moved = false;
  st = paged::tiles(a, &moved, s);
  if (st == SA_OK && paged::tile_tokens(a.rows, a.total, a.max_count) > 1) st = paged::decode(a, true, s);
  if (st != SA_OK && moved) {            // a call that fails leaves the histories as they were
    const int back = paged::restore_histories(a, s);
    if (back != SA_OK) return back;
  }
  return st;
}

unsigned long long sa_stream_capture(void* stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &id) != cudaSuccess) return ~0ull;
  return status == cudaStreamCaptureStatusNone ? 0 : id + 1;
}

size_t sa_beam_workspace_bytes(int dtype, int groups, int beams, int vocab, int width) {
  if (dtype < SA_F32 || dtype > SA_F16 || groups < 1 || beams < 1 || beams > beam::kMaxBeams || vocab < 1 || width < 1 ||
      width > beam::kMaxWidth || (int64_t)groups * beams > (1 << 20))
    return 0;
  return beam::workspace_bytes(dtype, groups, beams, vocab, width);
}

int sa_beam_select(const sa_beam* in) {
  if (in == nullptr || in->struct_bytes != (int32_t)sizeof(sa_beam)) return SA_ERR_BAD_ARGUMENT;
  if (in->dtype < SA_F32 || in->dtype > SA_F16 || in->groups < 1 || in->beams < 1 || in->vocab < 1 || in->width < 1) return SA_ERR_BAD_ARGUMENT;
  if (in->beams > beam::kMaxBeams || in->width > beam::kMaxWidth || (int64_t)in->width > (int64_t)in->beams * in->vocab)
    return SA_ERR_UNSUPPORTED;
  if ((int64_t)in->groups * in->beams > (1 << 20)) return SA_ERR_TOO_LARGE;
  if (!in->logits || !in->scores || !in->out_scores || !in->out_rows || !in->out_tokens || !in->workspace) return SA_ERR_BAD_ARGUMENT;
  if (!aligned(in->logits, in->dtype == SA_F32 ? 4 : 2) || !aligned(in->workspace, 16) || !aligned(in->out_tokens, 8)) return SA_ERR_ALIGNMENT;
  if (in->workspace_bytes < beam::workspace_bytes(in->dtype, in->groups, in->beams, in->vocab, in->width)) return SA_ERR_WORKSPACE;
  if (tc::timeout_pending()) return SA_ERR_DEVICE_TIMEOUT;
  const beam::Select p{in->dtype, in->groups, in->beams, in->vocab, in->width, in->logits, in->group_stride, in->beam_stride, in->scores,
                       in->out_scores, in->out_rows, reinterpret_cast<long long*>(in->out_tokens), in->workspace};
  return beam::select(p, static_cast<cudaStream_t>(in->stream));
}

}  // extern "C"
