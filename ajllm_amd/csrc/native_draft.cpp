// The operators of checking drafted tokens for the tensors they are nearly always called with, without the interpreter: one call of libajq_draft.so
// each, as in native_serve.cpp (None where anything is out of the ordinary).
#include "native_common.h"

#include "../../include/ajq_draft.h"

namespace native {
namespace {

decltype(&ajqt_tree_attention_workspace) tree_workspace;
decltype(&ajqt_tree_attention) run_tree;
decltype(&ajqt_keep_rows) run_keep;
decltype(&ajqt_log_probs_workspace) log_probs_workspace;
decltype(&ajqt_log_probs) run_log_probs;
decltype(&ajqt_follow_drafts) run_follow;

bool wrong_call(const char* what, bool bound, Py_ssize_t count, Py_ssize_t wanted) {
  if (count == wanted && bound) return false;
  if (count != wanted) PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", what, wanted);
  else PyErr_Format(PyExc_TypeError, "%s is not bound to the library", what);
  return true;
}
// elements from a row to the next (of a single row: any number that holds it)
int64_t apart(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
at::Tensor room_of(size_t bytes, const at::Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}
PyObject* wrap(at::Tensor t) {
  if (t.defined()) return THPVariable_Wrap(std::move(t));
  Py_RETURN_NONE;
}

}  // namespace

// (q, keys, values, rows, masks, counts, offset)
PyObject* tree_attention(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (wrong_call("tree_attention", run_tree, count, 7)) return nullptr;
  if (watched()) Py_RETURN_NONE;
  Arguments in{args};
  const at::Tensor *q = in.tensor(0), *keys = in.tensor(1), *values = in.tensor(2), *rows = in.tensor(3), *masks = in.tensor(4),
                   *counts = in.optional(5), *offset = in.optional(6);
  in.caches(keys, values);
  if (!in.ok || in.device != c10::hip::current_device()) Py_RETURN_NONE;
  in.need(q->dim() == 4 && Arguments::known(q->scalar_type()) && q->is_contiguous() && q->numel() > 0 && keys->size(0) == q->size(0) &&
          keys->size(3) == q->size(3) && fits(q->size(1)) && fits(q->size(2)));
  if (!in.ok) Py_RETURN_NONE;
  const int64_t batch = q->size(0), heads = q->size(1), nodes = q->size(2), hd = q->size(3), d = masks->dim();
  in.need((d == 2 || d == 3) && masks->scalar_type() == at::kInt && masks->size(d - 2) == nodes && masks->size(d - 1) >= (nodes + 31) / 32 &&
          masks->stride(d - 1) == 1 && (d == 2 || masks->size(0) == batch));
  ajqt_tree_attention_args a{};
  a.rows = in.whole(rows, batch);
  a.counts = in.whole(counts, batch);
  a.offset = in.whole(offset, 1);
  if (!in.ok) Py_RETURN_NONE;
  a.q = q->const_data_ptr();
  a.keys = keys->const_data_ptr();
  a.values = values->const_data_ptr();
  a.masks = reinterpret_cast<const uint32_t*>(masks->const_data_ptr<int32_t>());
  a.cache_batch = keys->stride(0);
  a.cache_head = keys->stride(1);
  a.mask_batch = d == 3 ? masks->stride(0) : 0;
  a.mask_token = masks->stride(d - 2);
  a.batch = as_int(batch);
  a.tokens = as_int(nodes);
  a.heads = as_int(heads);
  a.kv_heads = as_int(keys->size(1));
  a.dim = as_int(hd);
  a.max_len = as_int(keys->size(2));
  a.q_dtype = Arguments::flag(q->scalar_type());
  a.cache_dtype = Arguments::flag(keys->scalar_type());
  at::Tensor out;
  int status;
  {
    const WithoutInterpreter released;
    out = at::empty({batch, nodes, heads * hd}, q->options().dtype(at::kBFloat16));
    a.out = out.mutable_data_ptr();
    const size_t bytes = tree_workspace(&a);
    const at::Tensor room = room_of(bytes, *q);
    status = run_tree(&a, bytes ? room.mutable_data_ptr() : nullptr, bytes, c10::hip::getCurrentHIPStream(in.device).stream());
  }
  if (status != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (keys, values, rows, index, counts, offset); True where it is done
PyObject* keep_rows(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (wrong_call("keep_rows", run_keep, count, 6)) return nullptr;
  if (watched()) Py_RETURN_NONE;
  Arguments in{args};
  const at::Tensor *keys = in.tensor(0), *values = in.tensor(1), *rows = in.tensor(2), *index = in.tensor(3), *counts = in.optional(4),
                   *offset = in.optional(5);
  if (!in.ok || in.device != c10::hip::current_device()) Py_RETURN_NONE;
  const int64_t d = keys->dim(), n = index->dim();
  in.need((d == 4 || d == 5) && keys->sizes() == values->sizes() && keys->strides() == values->strides() && Arguments::known(keys->scalar_type()) &&
          values->scalar_type() == keys->scalar_type() && keys->numel() > 0);
  in.need(in.ok && keys->stride(d - 1) == 1 && keys->stride(d - 2) == keys->size(d - 1) && (n == 1 || n == 2) && index->scalar_type() == at::kLong && index->numel() > 0 &&
          (index->size(n - 1) == 1 || index->stride(n - 1) == 1) && fits(index->size(n - 1)));
  for (int i = 0; in.ok && i < d; ++i) in.need(fits(keys->size(i)));
  if (!in.ok) Py_RETURN_NONE;
  const int64_t batch = keys->size(d - 4);
  in.need(n == 1 || index->size(0) == batch);
  ajqt_keep_rows_args a{};
  a.rows = in.whole(rows, batch);
  a.counts = in.whole(counts, batch);
  a.offset = in.whole(offset, 1);
  if (!in.ok) Py_RETURN_NONE;
  a.index = index->const_data_ptr<int64_t>();
  a.keys = keys->mutable_data_ptr();
  a.values = values->mutable_data_ptr();
  a.cache_layer = d == 5 ? keys->stride(0) : 0;
  a.cache_batch = keys->stride(d - 4);
  a.cache_head = keys->stride(d - 3);
  a.index_ld = n == 2 ? index->stride(0) : 0;
  a.layers = d == 5 ? as_int(keys->size(0)) : 1;
  a.batch = as_int(batch);
  a.kv_heads = as_int(keys->size(d - 3));
  a.dim = as_int(keys->size(d - 1));
  a.max_len = as_int(keys->size(d - 2));
  a.width = as_int(index->size(n - 1));
  a.dtype = Arguments::flag(keys->scalar_type());
  int status;
  {
    const WithoutInterpreter released;
    status = run_keep(&a, c10::hip::getCurrentHIPStream(in.device).stream());
  }
  if (status != 0) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// (logits, targets, top): (log_probs, ranks, entropy, top_log_probs, top_ids)
PyObject* token_log_probs(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (wrong_call("token_log_probs", run_log_probs, count, 3)) return nullptr;
  if (watched()) Py_RETURN_NONE;
  Arguments in{args};
  const at::Tensor *logits = in.tensor(0), *targets = in.optional(1);
  const int64_t top = in.number(2);
  if (!in.ok || in.device != c10::hip::current_device()) Py_RETURN_NONE;
  in.need(logits->dim() == 2 && Arguments::known(logits->scalar_type()) && logits->numel() > 0 && (logits->size(1) == 1 || logits->stride(1) == 1) &&
          fits(logits->size(0)) && fits(logits->size(1)) && fits(top) && top <= logits->size(1));
  if (!in.ok) Py_RETURN_NONE;
  const int64_t rows = logits->size(0);
  in.need(targets == nullptr || targets->dim() == 1);
  ajqt_log_probs_args a{};
  a.targets = in.whole(targets, rows);
  if (!in.ok) Py_RETURN_NONE;
  a.logits = logits->const_data_ptr();
  a.ld = apart(*logits);
  a.rows = as_int(rows);
  a.vocab = as_int(logits->size(1));
  a.top = as_int(top);
  a.dtype = Arguments::flag(logits->scalar_type());
  at::Tensor log_probs, ranks, entropy, top_log_probs, top_ids;
  int status;
  {
    const WithoutInterpreter released;
    const auto floats = logits->options().dtype(at::kFloat), whole = logits->options().dtype(at::kLong);
    entropy = at::empty({rows}, floats);
    a.entropy = entropy.mutable_data_ptr<float>();
    if (targets) {
      log_probs = at::empty({rows}, floats);
      ranks = at::empty({rows}, whole);
      a.log_probs = log_probs.mutable_data_ptr<float>();
      a.ranks = ranks.mutable_data_ptr<int64_t>();
    }
    if (top) {
      top_log_probs = at::empty({rows, top}, floats);
      top_ids = at::empty({rows, top}, whole);
      a.top_log_probs = top_log_probs.mutable_data_ptr<float>();
      a.top_ids = top_ids.mutable_data_ptr<int64_t>();
    }
    const size_t bytes = log_probs_workspace(&a);
    const at::Tensor room = room_of(bytes, *logits);
    status = run_log_probs(&a, bytes ? room.mutable_data_ptr() : nullptr, bytes, c10::hip::getCurrentHIPStream(in.device).stream());
  }
  if (status != 0) Py_RETURN_NONE;
  PyObject* made[] = {wrap(std::move(log_probs)), wrap(std::move(ranks)), wrap(std::move(entropy)), wrap(std::move(top_log_probs)), wrap(std::move(top_ids))};
  PyObject* all = PyTuple_New(5);
  for (int i = 0; i < 5; ++i) {
    if (all) PyTuple_SET_ITEM(all, i, made[i]);
    else Py_XDECREF(made[i]);
  }
  return all;
  END_HANDLE_TH_ERRORS
}

// (tokens, parents, choices, counts): (path, accepted, chosen)
PyObject* follow_drafts(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (wrong_call("follow_drafts", run_follow, count, 4)) return nullptr;
  if (watched()) Py_RETURN_NONE;
  Arguments in{args};
  const at::Tensor *tokens = in.tensor(0), *parents = in.tensor(1), *choices = in.tensor(2), *counts = in.optional(3);
  if (!in.ok || in.device != c10::hip::current_device()) Py_RETURN_NONE;
  in.need(tokens->dim() == 2 && tokens->scalar_type() == at::kLong && tokens->numel() > 0 && (tokens->size(1) == 1 || tokens->stride(1) == 1) &&
          fits(tokens->size(0)) && fits(tokens->size(1)) && choices->scalar_type() == at::kLong && choices->sizes() == tokens->sizes() &&
          parents->scalar_type() == at::kLong);
  if (!in.ok) Py_RETURN_NONE;
  const int64_t batch = tokens->size(0), nodes = tokens->size(1), d = parents->dim();
  in.need((d == 1 || (d == 2 && parents->size(0) == batch)) && parents->size(d - 1) == nodes && (nodes == 1 || parents->stride(d - 1) == 1) &&
          (counts == nullptr || counts->dim() == 1));
  ajqt_follow_drafts_args a{};
  a.counts = in.whole(counts, batch);
  if (!in.ok) Py_RETURN_NONE;
  a.tokens = tokens->const_data_ptr<int64_t>();
  a.parents = parents->const_data_ptr<int64_t>();
  a.choices = choices->const_data_ptr<int64_t>();
  a.tokens_ld = tokens->stride(0);
  a.parents_ld = d == 2 ? parents->stride(0) : 0;
  a.choices_ld = choices->stride(0);
  a.choices_step = choices->stride(1);
  a.batch = as_int(batch);
  a.nodes = as_int(nodes);
  at::Tensor path, accepted, chosen;
  int status;
  {
    const WithoutInterpreter released;
    path = at::empty({batch, nodes}, tokens->options());
    accepted = at::empty({batch}, tokens->options());
    chosen = at::empty({batch, nodes}, tokens->options());
    a.path = path.mutable_data_ptr<int64_t>();
    a.accepted = accepted.mutable_data_ptr<int64_t>();
    a.chosen = chosen.mutable_data_ptr<int64_t>();
    status = run_follow(&a, c10::hip::getCurrentHIPStream(in.device).stream());
  }
  if (status != 0) Py_RETURN_NONE;
  PyObject* made[] = {wrap(std::move(path)), wrap(std::move(accepted)), wrap(std::move(chosen))};
  PyObject* all = PyTuple_New(3);
  for (int i = 0; i < 3; ++i) {
    if (all) PyTuple_SET_ITEM(all, i, made[i]);
    else Py_XDECREF(made[i]);
  }
  return all;
  END_HANDLE_TH_ERRORS
}

// bind_draft(tree_attention_workspace, tree_attention, keep_rows, log_probs_workspace, log_probs, follow_drafts): their addresses in the loaded library
PyObject* bind_draft(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 6) {
    PyErr_SetString(PyExc_TypeError, "bind_draft takes six addresses");
    return nullptr;
  }
  void* at[6];
  for (int i = 0; i < 6; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  tree_workspace = reinterpret_cast<decltype(tree_workspace)>(at[0]);
  run_tree = reinterpret_cast<decltype(run_tree)>(at[1]);
  run_keep = reinterpret_cast<decltype(run_keep)>(at[2]);
  log_probs_workspace = reinterpret_cast<decltype(log_probs_workspace)>(at[3]);
  run_log_probs = reinterpret_cast<decltype(run_log_probs)>(at[4]);
  run_follow = reinterpret_cast<decltype(run_follow)>(at[5]);
  Py_RETURN_NONE;
}

}  // namespace native
