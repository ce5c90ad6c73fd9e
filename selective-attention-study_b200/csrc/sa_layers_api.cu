// extern "C" boundary of what a decoder has around its attention: layer norm, the embedding, and the loss over a vocabulary.  Arguments
// are checked before anything is launched.
#include "sa_layers.cuh"
#include "sa_loss.cuh"
#include "sa_tc_host.cuh"

namespace sa {
namespace {

bool type_ok(int t) { return t == SA_F32 || t == SA_BF16 || t == SA_F16; }
bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
size_t bytes_of(int dtype) { return dtype == SA_F32 ? 4 : 2; }
bool fits(const void* p, int dtype) { return aligned(p, bytes_of(dtype)); }

int check_norm(const sa_norm* p, bool backward) {
  if (p == nullptr || p->struct_bytes != (int32_t)sizeof(sa_norm)) return SA_ERR_BAD_ARGUMENT;
  if (!type_ok(p->x_dtype) || !type_ok(p->branch_dtype) || !type_ok(p->y_dtype) || !type_ok(p->weight_dtype)) return SA_ERR_BAD_ARGUMENT;
  if (p->width < 1 || p->rows < 1 || !(p->eps >= 0.f) || p->x_stride < 0 || p->branch_stride < 0 || p->dy_stride < 0 || p->dsum_stride < 0)
    return SA_ERR_BAD_ARGUMENT;
  if (p->width > norm::kMaxWidth) return SA_ERR_UNSUPPORTED;
  if (p->rows > (1ll << 31) - 1) return SA_ERR_TOO_LARGE;
  if (p->x == nullptr) return SA_ERR_BAD_ARGUMENT;
  if (!fits(p->x, p->x_dtype) || !fits(p->branch, p->branch_dtype) || !fits(p->weight, p->weight_dtype) || !fits(p->bias, p->weight_dtype) ||
      !aligned(p->stats, 4))
    return SA_ERR_ALIGNMENT;
  if (!backward) {
    if (p->y == nullptr || (p->branch != nullptr) != (p->sum != nullptr)) return SA_ERR_BAD_ARGUMENT;
    return fits(p->sum, p->x_dtype) && fits(p->y, p->y_dtype) ? SA_OK : SA_ERR_ALIGNMENT;
  }
  if (p->dy == nullptr || p->dx == nullptr || p->stats == nullptr) return SA_ERR_BAD_ARGUMENT;
  if (p->dweight != nullptr && p->weight == nullptr) return SA_ERR_BAD_ARGUMENT;
  if (!fits(p->dy, p->y_dtype) || !fits(p->dsum, p->x_dtype) || !fits(p->dx, p->x_dtype) || !fits(p->dbranch, p->branch_dtype) ||
      !fits(p->dweight, p->weight_dtype) || !fits(p->dbias, p->weight_dtype))
    return SA_ERR_ALIGNMENT;
  return SA_OK;
}

int check_embedding(const sa_embedding* p, bool backward) {
  if (p == nullptr || p->struct_bytes != (int32_t)sizeof(sa_embedding)) return SA_ERR_BAD_ARGUMENT;
  if (!type_ok(p->weight_dtype) || !type_ok(p->y_dtype)) return SA_ERR_BAD_ARGUMENT;
  if (p->tokens < 1 || p->vocab < 1 || p->width < 1 || p->weight_stride < 0 || p->dy_stride < 0) return SA_ERR_BAD_ARGUMENT;
  if (p->tokens > (1 << 30) || p->vocab > (1 << 30) || p->width > (1 << 20)) return SA_ERR_TOO_LARGE;
  if (p->idx == nullptr || !aligned(p->idx, 8)) return p->idx == nullptr ? SA_ERR_BAD_ARGUMENT : SA_ERR_ALIGNMENT;
  const void* const in = backward ? p->dy : p->weight;
  const void* const out = backward ? p->dweight : p->y;
  if (in == nullptr || out == nullptr) return SA_ERR_BAD_ARGUMENT;
  const bool ok = backward ? fits(in, p->y_dtype) && fits(out, p->weight_dtype) : fits(in, p->weight_dtype) && fits(out, p->y_dtype);
  return ok ? SA_OK : SA_ERR_ALIGNMENT;
}

int to_loss(const sa_linear_loss* in, loss::Problem* p) {
  if (in == nullptr || in->struct_bytes != (int32_t)sizeof(sa_linear_loss)) return SA_ERR_BAD_ARGUMENT;
  if (!type_ok(in->product) || !type_ok(in->x_dtype) || !type_ok(in->weight_dtype)) return SA_ERR_BAD_ARGUMENT;
  if (in->reduction < SA_REDUCTION_NONE || in->reduction > SA_REDUCTION_MEAN) return SA_ERR_BAD_ARGUMENT;
  if (in->tokens < 1 || in->vocab < 1 || in->width < 1 || in->x_stride < 0 || in->weight_stride < 0) return SA_ERR_BAD_ARGUMENT;
  if (in->tokens > (1 << 24) || in->vocab > (1 << 24) || in->width > (1 << 16)) return SA_ERR_TOO_LARGE;
  // sums of 24-bit products are kept in fp32 only where results are
  if (in->product == SA_F32 && (in->x_dtype != SA_F32 || in->weight_dtype != SA_F32)) return SA_ERR_UNSUPPORTED;
  *p = loss::Problem{in->product, in->x_dtype, in->weight_dtype, in->reduction, in->tokens, in->vocab, in->width, in->ignore_index, in->x, in->x_stride,
                     in->weight, in->weight_stride, in->targets, in->lse, in->count, in->loss, in->dloss, in->dx, in->dweight, in->dx_sums, in->dweight_sums,
                     in->workspace};
  return SA_OK;
}

// The form that computes the gradients with the loss: one cotangent, and operands whose exponents hold e^44.
int check_train(const sa_linear_loss* in) {
  if (in->reduction == SA_REDUCTION_NONE || in->product == SA_F16) return SA_ERR_UNSUPPORTED;
  if (!in->dx_sums && !in->dweight_sums) return SA_ERR_BAD_ARGUMENT;
  return aligned(in->dx_sums, 4) && aligned(in->dweight_sums, 4) ? SA_OK : SA_ERR_ALIGNMENT;
}

int check_loss(const sa_linear_loss* in, bool backward, size_t need) {
  if (!in->x || !in->weight || !in->targets || !in->lse || !in->workspace) return SA_ERR_BAD_ARGUMENT;
  if (in->reduction != SA_REDUCTION_NONE && !in->count) return SA_ERR_BAD_ARGUMENT;
  if (backward ? !in->dloss || (!in->dx && !in->dweight) : !in->loss) return SA_ERR_BAD_ARGUMENT;
  if (!fits(in->x, in->x_dtype) || !fits(in->weight, in->weight_dtype) || !aligned(in->targets, 8) || !aligned(in->lse, 8) || !aligned(in->count, 4) ||
      !aligned(in->loss, 4) || !aligned(in->dloss, 4) || !fits(in->dx, in->x_dtype) || !fits(in->dweight, in->weight_dtype) ||
      !aligned(in->workspace, 256))
    return SA_ERR_ALIGNMENT;
  if (in->workspace_bytes < need) return SA_ERR_WORKSPACE;
  return tc::timeout_pending() ? SA_ERR_DEVICE_TIMEOUT : SA_OK;
}

}  // namespace
}  // namespace sa

using namespace sa;

extern "C" {

int sa_norm_forward(const sa_norm* p) {
  const int st = check_norm(p, false);
  return st != SA_OK ? st : norm::forward(*p, static_cast<cudaStream_t>(p->stream));
}

size_t sa_norm_backward_bytes(const sa_norm* p) {
  if (p == nullptr || p->struct_bytes != (int32_t)sizeof(sa_norm) || p->width < 1 || p->width > norm::kMaxWidth || p->rows < 1) return 0;
  return norm::backward_bytes(*p);
}

int sa_norm_backward(const sa_norm* p) {
  const int st = check_norm(p, true);
  if (st != SA_OK) return st;
  const size_t need = norm::backward_bytes(*p);
  if (need > 0 && p->workspace == nullptr) return SA_ERR_BAD_ARGUMENT;
  if (need > 0 && !aligned(p->workspace, 16)) return SA_ERR_ALIGNMENT;
  if (p->workspace_bytes < need) return SA_ERR_WORKSPACE;
  if (tc::timeout_pending()) return SA_ERR_DEVICE_TIMEOUT;
  return norm::backward(*p, static_cast<cudaStream_t>(p->stream));
}

int sa_embedding_forward(const sa_embedding* p) {
  const int st = check_embedding(p, false);
  return st != SA_OK ? st : embed::forward(*p, static_cast<cudaStream_t>(p->stream));
}

size_t sa_embedding_backward_bytes(const sa_embedding* p) {
  if (p == nullptr || p->struct_bytes != (int32_t)sizeof(sa_embedding) || p->tokens < 1 || p->vocab < 1 || p->width < 1) return 0;
  return embed::backward_bytes(*p);
}

int sa_embedding_backward(const sa_embedding* p) {
  const int st = check_embedding(p, true);
  if (st != SA_OK) return st;
  if (p->workspace == nullptr) return SA_ERR_BAD_ARGUMENT;
  if (!aligned(p->workspace, 16)) return SA_ERR_ALIGNMENT;
  if (p->workspace_bytes < embed::backward_bytes(*p)) return SA_ERR_WORKSPACE;
  return embed::backward(*p, static_cast<cudaStream_t>(p->stream));
}

size_t sa_linear_loss_forward_bytes(const sa_linear_loss* in) {
  loss::Problem p;
  return to_loss(in, &p) == SA_OK ? loss::forward_bytes(p) : 0;
}

int sa_linear_loss_forward(const sa_linear_loss* in) {
  loss::Problem p;
  int st = to_loss(in, &p);
  if (st == SA_OK) st = check_loss(in, false, loss::forward_bytes(p));
  return st != SA_OK ? st : loss::forward(p, static_cast<cudaStream_t>(in->stream));
}

size_t sa_linear_loss_backward_bytes(const sa_linear_loss* in) {
  loss::Problem p;
  return to_loss(in, &p) == SA_OK ? loss::backward_bytes(p) : 0;
}

int sa_linear_loss_backward(const sa_linear_loss* in) {
  loss::Problem p;
  int st = to_loss(in, &p);
  if (st == SA_OK) st = check_loss(in, true, loss::backward_bytes(p));
  return st != SA_OK ? st : loss::backward(p, static_cast<cudaStream_t>(in->stream));
}

int sa_linear_loss_prefers_train(const sa_linear_loss* in) {
  loss::Problem p;
  return to_loss(in, &p) == SA_OK && loss::prefers_train(p);
}

size_t sa_linear_loss_train_bytes(const sa_linear_loss* in) {
  loss::Problem p;
  return to_loss(in, &p) == SA_OK && check_train(in) == SA_OK ? loss::train_bytes(p) : 0;
}

int sa_linear_loss_train(const sa_linear_loss* in) {
  loss::Problem p;
  int st = to_loss(in, &p);
  if (st == SA_OK) st = check_train(in);
  if (st != SA_OK) return st;
  if (!in->x || !in->weight || !in->targets || !in->count || !in->loss || !in->workspace) return SA_ERR_BAD_ARGUMENT;
  if (!fits(in->x, in->x_dtype) || !fits(in->weight, in->weight_dtype) || !aligned(in->targets, 8) || !aligned(in->count, 4) ||
      !aligned(in->loss, 4) || !aligned(in->workspace, 256))
    return SA_ERR_ALIGNMENT;
  if (in->workspace_bytes < loss::train_bytes(p)) return SA_ERR_WORKSPACE;
  return tc::timeout_pending() ? SA_ERR_DEVICE_TIMEOUT : loss::train(p, static_cast<cudaStream_t>(in->stream));
}

int sa_linear_loss_scale(const sa_linear_loss* in) {
  loss::Problem p;
  int st = to_loss(in, &p);
  if (st == SA_OK) st = check_train(in);
  if (st != SA_OK) return st;
  if (!in->dloss || !in->count || (!in->dx && !in->dweight) || (in->dx && !in->dx_sums) || (in->dweight && !in->dweight_sums)) return SA_ERR_BAD_ARGUMENT;
  if (!aligned(in->dloss, 4) || !aligned(in->count, 4) || !fits(in->dx, in->x_dtype) || !fits(in->dweight, in->weight_dtype)) return SA_ERR_ALIGNMENT;
  return loss::scale(p, static_cast<cudaStream_t>(in->stream));
}

}  // extern "C"
