// The operators of decoding many continuations of one prompt for the tensors they are nearly always called with, without the interpreter: one
// call of libajq_serve.so each.
//
// Every function returns None where anything is out of the ordinary (a dtype, shape or layout that the package's function refuses or
// converts, a subclass, a mode that wants to see the operators, another device than the current one, an error status): the
// caller then goes through its general path.  What bounds a decode step's calls is the host: 14 to 16 us through ctypes, where the kernels
// take 3 to 5.
#include "native_common.h"

#include "../../include/ajq_serve.h"

namespace native {
namespace {

decltype(&ajqs_norm_rope) run_norm_rope;
decltype(&ajqs_shared_attention_workspace) attention_workspace;
decltype(&ajqs_shared_attention) run_attention;
decltype(&ajqs_adjust_logits) run_adjust;

// Reads a call's arguments one after the other; `ok` falls at the first that is not as expected.
struct Arguments {
  PyObject* const* args;
  c10::DeviceIndex device = -1;
  bool ok = true;
  at::Tensor held[16];   // references, while the interpreter runs other threads
  int holds = 0;

  const at::Tensor* tensor(int i) {
    if (!ok) return nullptr;
    const at::Tensor* t = plain(args[i]);
    if (t == nullptr || (device >= 0 && t->device().index() != device)) {
      ok = false;
      return nullptr;
    }
    device = t->device().index();
    held[holds] = *t;
    return &held[holds++];
  }
  const at::Tensor* optional(int i) { return args[i] == Py_None ? nullptr : tensor(i); }
  int64_t number(int i) {
    if (!ok || !PyLong_CheckExact(args[i])) {
      ok = false;
      return 0;
    }
    const int64_t n = PyLong_AsLongLong(args[i]);
    if (n == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return n;
  }
  void need(bool condition) { ok = ok && condition; }

  static bool known(at::ScalarType type) { return type == at::kFloat || type == at::kBFloat16; }
  static int flag(at::ScalarType type) { return type == at::kBFloat16 ? AJQS_BF16 : AJQS_F32; }
  // int64, contiguous, `count` of them
  const int64_t* whole(const at::Tensor* t, int64_t count) {
    if (!ok || t == nullptr) return nullptr;
    need(t->scalar_type() == at::kLong && t->numel() == count && t->is_contiguous());
    return ok ? t->const_data_ptr<int64_t>() : nullptr;
  }
  const float* floats(const at::Tensor* t, at::IntArrayRef shape) {
    if (!ok || t == nullptr) return nullptr;
    need(t->scalar_type() == at::kFloat && t->sizes() == shape && t->is_contiguous());
    return ok ? t->const_data_ptr<float>() : nullptr;
  }
  void caches(const at::Tensor* keys, const at::Tensor* values) {
    if (!ok) return;
    need(keys->dim() == 4 && keys->sizes() == values->sizes() && keys->strides() == values->strides() && known(keys->scalar_type()) &&
         values->scalar_type() == keys->scalar_type());
    need(ok && keys->stride(3) == 1 && keys->stride(2) == keys->size(3));
    for (int d = 0; ok && d < 4; ++d) need(keys->size(d) >= 1 && keys->size(d) <= INT32_MAX);
  }
};

int as_int(int64_t n) { return (int)n; }
bool fits(int64_t n) { return n >= 0 && n <= INT32_MAX; }

}  // namespace

// (qkv, cosine, sine, keys, values, rows, heads, tokens, q_gain, k_gain, epsilon, positions, counts, offset, out_dtype)
PyObject* norm_rope(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 15 || !run_norm_rope) {
    PyErr_SetString(PyExc_TypeError, count != 15 ? "norm_rope takes fifteen arguments" : "norm_rope is not bound to the library");
    return nullptr;
  }
  if (watched()) Py_RETURN_NONE;
  Arguments in{args};
  const at::Tensor *qkv = in.tensor(0), *cosine = in.tensor(1), *sine = in.tensor(2), *keys = in.tensor(3), *values = in.tensor(4),
                   *rows = in.tensor(5), *q_gain = in.optional(8), *k_gain = in.optional(9), *positions = in.optional(11),
                   *counts = in.optional(12), *offset = in.optional(13);
  const int64_t heads = in.number(6), tokens = in.number(7);
  in.need(PyFloat_CheckExact(args[10]) && THPDtype_Check(args[14]));
  in.caches(keys, values);
  if (!in.ok || in.device != c10::hip::current_device()) Py_RETURN_NONE;
  const at::ScalarType type = reinterpret_cast<THPDtype*>(args[14])->scalar_type;
  const int64_t batch = keys->size(0), kv_heads = keys->size(1), hd = keys->size(3);
  in.need(Arguments::known(type) && Arguments::known(qkv->scalar_type()) && qkv->dim() == 2 && fits(heads) && fits(tokens) && heads <= 1 << 20 &&
          kv_heads <= 1 << 20 && hd <= 1 << 10 && fits(batch * tokens) && qkv->size(0) == batch * tokens &&
          qkv->size(1) == (heads + 2 * kv_heads) * hd && (qkv->numel() == 0 || qkv->stride(1) == 1) && cosine->dim() == 2 && fits(cosine->size(0)));
  if (!in.ok) Py_RETURN_NONE;
  const int64_t table[2] = {cosine->size(0), hd / 2}, gain[1] = {hd};
  ajqs_norm_rope_args a{};
  a.qkv = qkv->const_data_ptr();
  a.cosine = in.floats(cosine, table);
  a.sine = in.floats(sine, table);
  a.q_gain = in.floats(q_gain, gain);
  a.k_gain = in.floats(k_gain, gain);
  a.rows = in.whole(rows, batch);
  a.positions = in.whole(positions, batch);
  a.counts = in.whole(counts, batch);
  a.offset = in.whole(offset, 1);
  if (!in.ok) Py_RETURN_NONE;
  a.keys = keys->mutable_data_ptr();
  a.values = values->mutable_data_ptr();
  a.ld = qkv->stride(0);
  a.cache_batch = keys->stride(0);
  a.cache_head = keys->stride(1);
  a.batch = as_int(batch);
  a.tokens = as_int(tokens);
  a.heads = as_int(heads);
  a.kv_heads = as_int(kv_heads);
  a.dim = as_int(hd);
  a.max_len = as_int(keys->size(2));
  a.table_rows = as_int(cosine->size(0));
  a.in_dtype = Arguments::flag(qkv->scalar_type());
  a.q_dtype = Arguments::flag(type);
  a.cache_dtype = Arguments::flag(keys->scalar_type());
  a.eps = (float)PyFloat_AS_DOUBLE(args[10]);
  at::Tensor q;
  int status;
  {
    const WithoutInterpreter released;
    q = at::empty({batch, heads, tokens, hd}, qkv->options().dtype(type));
    a.q = q.mutable_data_ptr();
    status = run_norm_rope(&a, c10::hip::getCurrentHIPStream(in.device).stream());
  }
  if (status != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(q));
  END_HANDLE_TH_ERRORS
}

// (q, prefix_keys, prefix_values, prefix_lengths, keys, values, rows, counts, offset)
PyObject* shared_prefix_attention(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 9 || !run_attention) {
    PyErr_SetString(PyExc_TypeError, count != 9 ? "shared_prefix_attention takes nine arguments" : "shared_prefix_attention is not bound to the library");
    return nullptr;
  }
  if (watched()) Py_RETURN_NONE;
  Arguments in{args};
  const at::Tensor *q = in.tensor(0), *prefix_keys = in.tensor(1), *prefix_values = in.tensor(2), *lengths = in.tensor(3), *keys = in.tensor(4),
                   *values = in.tensor(5), *rows = in.tensor(6), *counts = in.optional(7), *offset = in.optional(8);
  in.caches(prefix_keys, prefix_values);
  in.caches(keys, values);
  if (!in.ok || in.device != c10::hip::current_device()) Py_RETURN_NONE;
  in.need(q->dim() == 4 && Arguments::known(q->scalar_type()) && q->is_contiguous() && q->numel() > 0 && keys->size(0) == q->size(0) &&
          keys->size(1) == prefix_keys->size(1) && keys->size(3) == q->size(3) && prefix_keys->size(3) == q->size(3) &&
          keys->scalar_type() == prefix_keys->scalar_type() && fits(q->size(1)) && fits(q->size(2)));
  if (!in.ok) Py_RETURN_NONE;
  const int64_t batch = q->size(0), heads = q->size(1), seq = q->size(2), hd = q->size(3);
  ajqs_shared_attention_args a{};
  a.prefix_lengths = in.whole(lengths, prefix_keys->size(0));
  a.rows = in.whole(rows, batch);
  a.counts = in.whole(counts, batch);
  a.offset = in.whole(offset, 1);
  if (!in.ok) Py_RETURN_NONE;
  a.q = q->const_data_ptr();
  a.prefix_keys = prefix_keys->const_data_ptr();
  a.prefix_values = prefix_values->const_data_ptr();
  a.keys = keys->const_data_ptr();
  a.values = values->const_data_ptr();
  a.prefix_group = prefix_keys->stride(0);
  a.prefix_head = prefix_keys->stride(1);
  a.cache_batch = keys->stride(0);
  a.cache_head = keys->stride(1);
  a.groups = as_int(prefix_keys->size(0));
  a.batch = as_int(batch);
  a.tokens = as_int(seq);
  a.heads = as_int(heads);
  a.kv_heads = as_int(keys->size(1));
  a.dim = as_int(hd);
  a.prefix_cap = as_int(prefix_keys->size(2));
  a.max_len = as_int(keys->size(2));
  a.q_dtype = Arguments::flag(q->scalar_type());
  a.cache_dtype = Arguments::flag(keys->scalar_type());
  at::Tensor out;
  int status;
  {
    const WithoutInterpreter released;
    out = at::empty({batch, seq, heads * hd}, q->options().dtype(at::kBFloat16));
    a.out = out.mutable_data_ptr();
    const size_t bytes = attention_workspace(&a);
    at::Tensor room;
    if (bytes) room = at::empty({(int64_t)bytes}, q->options().dtype(at::kByte));
    status = run_attention(&a, bytes ? room.mutable_data_ptr() : nullptr, bytes, c10::hip::getCurrentHIPStream(in.device).stream());
  }
  if (status != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (logits, tokens, lengths, prompt, prompt_lengths, repetition, frequency, presence, bias_ids, bias, allowed, allowed_rows, out)
PyObject* adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 13 || !run_adjust) {
    PyErr_SetString(PyExc_TypeError, count != 13 ? "adjust_logits takes thirteen arguments" : "adjust_logits is not bound to the library");
    return nullptr;
  }
  if (watched()) Py_RETURN_NONE;
  Arguments in{args};
  const at::Tensor *logits = in.tensor(0), *tokens = in.optional(1), *lengths = in.optional(2), *prompt = in.optional(3),
                   *prompt_lengths = in.optional(4), *repetition = in.optional(5), *frequency = in.optional(6), *presence = in.optional(7),
                   *bias_ids = in.optional(8), *bias = in.optional(9), *allowed = in.optional(10), *allowed_rows = in.optional(11),
                   *given = in.optional(12);
  if (!in.ok || in.device != c10::hip::current_device()) Py_RETURN_NONE;
  in.need(logits->dim() == 2 && Arguments::known(logits->scalar_type()) && logits->numel() > 0 && logits->stride(1) == 1 && fits(logits->size(0)) &&
          logits->size(1) <= INT32_MAX - 4 && (bias == nullptr) == (bias_ids == nullptr) && (lengths == nullptr || tokens != nullptr) &&
          (prompt_lengths == nullptr || prompt != nullptr) && (allowed_rows == nullptr || allowed != nullptr));
  if (!in.ok) Py_RETURN_NONE;
  const int64_t batch = logits->size(0), vocab = logits->size(1), of_rows[1] = {batch};
  // elements from a row to the next (of a single row: any number that holds it)
  auto apart = [](const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); };
  ajqs_adjust_logits_args a{};
  auto list = [&](const at::Tensor* ids, const at::Tensor* counts, const int64_t*& to, const int64_t*& count_to, int64_t& ld, int& most, int& stride) {
    if (!in.ok || ids == nullptr) return;
    in.need(ids->dim() == 2 && ids->size(0) == batch && ids->scalar_type() == at::kLong && fits(ids->size(1)) &&
            (ids->size(1) == 0 || ids->stride(1) == 1));
    if (counts) in.need(counts->scalar_type() == at::kLong && (counts->numel() == 1 || counts->numel() == batch) && counts->is_contiguous());
    if (!in.ok || ids->size(1) == 0) return;
    to = ids->const_data_ptr<int64_t>();
    count_to = counts ? counts->const_data_ptr<int64_t>() : nullptr;
    ld = apart(*ids);
    most = as_int(ids->size(1));
    stride = counts && counts->numel() == batch && batch > 1;
  };
  list(tokens, lengths, a.tokens, a.token_counts, a.tokens_ld, a.max_tokens, a.token_count_stride);
  list(prompt, prompt_lengths, a.prompt, a.prompt_counts, a.prompt_ld, a.max_prompt, a.prompt_count_stride);
  a.repetition = in.floats(repetition, of_rows);
  a.frequency = in.floats(frequency, of_rows);
  a.presence = in.floats(presence, of_rows);
  if (in.ok && bias) {
    in.need(bias->dim() == 2 && bias->size(0) == batch && bias_ids->sizes() == bias->sizes() && bias->scalar_type() == at::kFloat &&
            bias_ids->scalar_type() == at::kLong && bias->is_contiguous() && bias_ids->is_contiguous() && fits(bias->size(1)));
    if (!in.ok) Py_RETURN_NONE;
    a.bias_ids = bias_ids->const_data_ptr<int64_t>();
    a.bias = bias->const_data_ptr<float>();
    a.bias_ld = a.biases = as_int(bias->size(1));
  }
  if (in.ok && allowed) {
    in.need(allowed->dim() == 2 && allowed->scalar_type() == at::kInt && allowed->numel() > 0 && allowed->stride(1) == 1 &&
            fits(allowed->size(0)) && allowed->size(1) >= (vocab + 31) / 32);
    if (!in.ok) Py_RETURN_NONE;
    a.allowed = reinterpret_cast<const uint32_t*>(allowed->const_data_ptr<int32_t>());
    a.allowed_ld = apart(*allowed);
    a.masks = as_int(allowed->size(0));
    if (allowed_rows) {
      in.need(allowed_rows->dim() == 1);
      a.allowed_rows = in.whole(allowed_rows, batch);
    }
  }
  if (in.ok && given) in.need(given->sizes() == logits->sizes() && given->scalar_type() == at::kFloat && given->stride(1) == 1);
  if (!in.ok) Py_RETURN_NONE;
  a.logits = logits->const_data_ptr();
  a.ld = apart(*logits);
  a.batch = as_int(batch);
  a.vocab = as_int(vocab);
  a.dtype = Arguments::flag(logits->scalar_type());
  at::Tensor out;
  int status;
  {
    const WithoutInterpreter released;
    if (given) {
      out = *given;
    } else {
      const int64_t width = (vocab + 3) / 4 * 4;
      out = at::empty({batch, width}, logits->options().dtype(at::kFloat));
      if (width != vocab) out = out.narrow(1, 0, vocab);
    }
    a.out = out.mutable_data_ptr<float>();
    a.out_ld = apart(out);
    status = run_adjust(&a, c10::hip::getCurrentHIPStream(in.device).stream());
  }
  if (status != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// bind_serve(norm_rope, shared_attention_workspace, shared_attention, adjust_logits): their addresses in the loaded library
PyObject* bind_serve(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 4) {
    PyErr_SetString(PyExc_TypeError, "bind_serve takes four addresses");
    return nullptr;
  }
  void* at[4];
  for (int i = 0; i < 4; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  run_norm_rope = reinterpret_cast<decltype(run_norm_rope)>(at[0]);
  attention_workspace = reinterpret_cast<decltype(attention_workspace)>(at[1]);
  run_attention = reinterpret_cast<decltype(run_attention)>(at[2]);
  run_adjust = reinterpret_cast<decltype(run_adjust)>(at[3]);
  Py_RETURN_NONE;
}

}  // namespace native
