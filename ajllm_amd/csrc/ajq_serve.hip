// C ABI of libajq_serve.so (include/ajq_serve.h): argument validation, launch geometry, error reporting.
#include "serve_host.h"

#include "logits_kernels.h"
#include "norm_rope_kernels.h"
#include "shared_attention.h"

namespace {

constexpr int kMostRows = 1 << 30;   // of a cache head
int check_shared(const ajqs_shared_attention_args* a) {
  const char* what = "ajqs_shared_attention";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->q || !a->prefix_keys || !a->prefix_values || !a->keys || !a->values || !a->prefix_lengths || !a->rows || !a->out)
    return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (!built_dim(a->dim)) return fail(AJQ_ERR_UNSUPPORTED, "%s: head size %d (128, 64 and 32 are built)", what, a->dim);
  if (a->batch < 1 || a->tokens < 1 || a->groups < 1 || a->batch % a->groups != 0 || a->kv_heads < 1 || a->heads < 1 ||
      a->heads % a->kv_heads != 0 || a->prefix_cap < 1 || a->max_len < 1 || a->prefix_cap > kMostRows || a->max_len > kMostRows)
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (groups=%d batch=%d tokens=%d heads=%d kv_heads=%d prefix_cap=%d max_len=%d)", what,
                a->groups, a->batch, a->tokens, a->heads, a->kv_heads, a->prefix_cap, a->max_len);
  if ((long long)a->batch * a->heads * a->tokens > 0x1FFFFFFFLL)
    return fail(AJQ_ERR_SHAPE, "%s: too many queries (%d x %d x %d)", what, a->batch, a->heads, a->tokens);
  if (!known(a->q_dtype) || !known(a->cache_dtype)) return fail(AJQ_ERR_UNSUPPORTED, "%s: unknown element type", what);
  if (!aligned16(a->q) || !aligned16(a->out)) return fail(AJQ_ERR_ALIGN, "%s: q and out must be 16-byte aligned", what);
  if (int e = check_caches(what, a->prefix_keys, a->prefix_values, a->prefix_group, a->prefix_head)) return e;
  return check_caches(what, a->keys, a->values, a->cache_batch, a->cache_head);
}

// How an attention call is cut up: tiles of queries, parts of the rows.  The device's lengths are not known here; the capacities are what they
// can be.
enum class SharedForm { few, many, walk, each };   // (the prefix by meet_few, by meet_many; everything in one walk of many, of few queries)
struct SharedPlan {
  SharedForm form;
  int prefix_rt, own_rt;            // tiles of 16 queries a wave
  bool own_alone;                   // a wave a tile of own queries, not a workgroup
  int prefix_tiles, own_tiles, prefix_parts, own_parts;
  long long prefix_blocks, own_blocks, queries;
  size_t bytes;
};
constexpr int kMostParts = 64;      // a lane each in the merge
// Whether one launch in which every sequence walks the prefix by itself is the faster (sum of kernel times, against those of two launches; 32 / 8 heads of 128,
// bf16, rows of prefix + own): 8 sequences of 64 rows 4.7 and 9.0 us, of 512 6.7 and 9.4, of 768 7.7 and 9.2, of 1536 11.5 and 11.5; 128 sequences of 64 9.0 and
// 14.2, of 768 22.3 and 23.5, of 1536 49 and 39.  fp32 rows take longer in fp32: 8 of 64 6.3 and 11.2, of 192 8.5 and 11.5, of 512 14.4 and 12.9; 128 of 192 27.0
// and 28.8.
// With more of them than 1024, each to a wave (below): 4096 of 50 rows 12.6 and 17.1, 1536 of 130 10.1 and 11.8, of 260 14.1 and 12.9.
bool shared_each(const ajqs_shared_attention_args* a, long long tiles) {
  const long long rows = (long long)a->prefix_cap + a->max_len;
  if (a->cache_dtype == AJQS_BF16) return rows <= (tiles <= 1024 ? 768 : 128);
  return rows <= (tiles <= 1024 ? 192 : 64);
}
// Whether a wave takes a tile of a sequence's queries by itself, with the `rows` rows that they meet: no join, four times as many at once, but the longest is one
// wave's.  Behind a prefix, 1536 heads (128 sequences of 12 heads of 64) of 60 rows 9.9 and 13.5 us, of 200 16.6 and 17.4; of 128, of 300 rows 49.4 and 44.6;
// 512 (64 of 8) of 60 18.4 and 18.7.  Everything in one walk: 768 of 130 rows 7.7 and 9.6, of 430 14.9 and 14.7; 512 of 130 7.7 and 6.5.
bool shared_alone(long long tiles, long long rows, long long most) { return tiles >= 768 && rows <= most; }
SharedPlan shared_plan(const ajqs_shared_attention_args* a) {
  SharedPlan p{};
  const long long share = a->heads / a->kv_heads, mine = a->tokens * share, all = a->batch / a->groups * mine;
  const long long own_units = (long long)a->batch * a->kv_heads, prefix_units = (long long)a->groups * a->kv_heads;
  const bool bf16 = a->cache_dtype == AJQS_BF16;
  // parts of at least `least` rows, until there are `wanted` workgroups
  auto parts = [](long long workgroups, long long wanted, long long rows, long long least, long long most) {
    return (int)std::max(1ll, std::min({wanted / workgroups, ceil_div(rows, least), most}));
  };
  p.queries = (long long)a->batch * a->heads * a->tokens;
  if (bf16 && mine > 64) {
    p.form = SharedForm::walk;
    // Tiles of 128 queries (bf16 ones of 128 components: more do not leave registers, narrower heads' steps are too short) where there are enough of them and
    // most rows are the prefix's; else of 64.  (Both sides in first calls after a pause, whose clock is some 10 % lower.)  16 sequences of 100 tokens x 4 behind 2048 rows 74 us, 90 with tiles of 64; of 400 behind 2048 229 and 292; of 100
    // behind 100 + 1400 74 and 47; 8 of 40 behind 1000 24 and 21; 12 heads of 64, 16 of 300 behind 2048: 68 and 58.
    p.own_rt = a->q_dtype == AJQS_BF16 && a->dim == 128 && a->prefix_cap >= a->max_len && own_units * ceil_div(mine, 128) >= 256 ? 2 : 1;
    p.own_tiles = (int)ceil_div(mine, 64 * p.own_rt);
    p.own_parts = parts(own_units * p.own_tiles, 512, (long long)a->prefix_cap + a->max_len, 128, kMostParts);
    p.own_blocks = ceil_div(own_units, 8) * 8 * p.own_tiles * p.own_parts;
  } else if (shared_each(a, own_units * ceil_div(mine, 16))) {
    p.form = SharedForm::each;   // (always tiles of 16: 8 sequences of 7 tokens x 4 behind 500 rows with 250 8.9 us, of 32 13.1)
    p.own_rt = 1;
    p.own_tiles = (int)ceil_div(mine, 16);
    p.own_parts = 1;
    p.own_alone = shared_alone(own_units * p.own_tiles, (long long)a->prefix_cap + a->max_len, 384);
    p.own_blocks = p.own_alone ? ceil_div(own_units * p.own_tiles, 4) : ceil_div(own_units, 8) * 8 * p.own_tiles;
  } else {
    // 128 queries a head behind 8192 rows of 8 heads: few 21.9, many 22.3 us; 120 of 16 heads behind 4096 25.6 and 27.6; 256 behind 8192 31.0 and 27.9.  Behind 32768
    // rows of 8 heads, 64 queries 37.3 and 36.4, 96 50.2 and 43.7, 128 56.4 and 49.5; 96 of 16 heads behind 8192 44.1 and 47.4.
    p.form = bf16 && (all > 128 || (all > 64 && prefix_units * ceil_div(a->prefix_cap, 128) > 1024)) ? SharedForm::many : SharedForm::few;
    // Tiles of 32 queries fetch rows half as often as tiles of 16, which are twice as many and wait less: 16 it is while rows come from L2 and workgroups are few.  The
    // prefix (32 heads in five groups of 30 queries, 4672 fp32 rows: 137 us with 32, 221 with 16; 16 heads, 30 queries, 4000 rows 29.6 and 26.4; 8 heads, 64 queries,
    // 4000 bf16 rows 11.0 and 10.1, 64 fp32 19.6 and 21.5); own rows that are fp32 (64 sequences of 28 queries, 1000 rows 128 and 142 us; 2 of 28, 300 rows 23.4 and
    // 20.4).  bf16 own rows gain either way (8 of 24, 600 rows 15.9 and 13.6; 64 of 28, 1000 rows 53.6 and 54.2; 128 of 20, 1000 rows 72 and 79): always 16.
    auto tiles_of = [&](long long queries, long long units, long long rows, long long from_l2) {
      return queries > (units * ceil_div(rows, 128) > 512 ? 16 : from_l2) ? 2 : 1;
    };
    p.own_rt = bf16 ? 1 : tiles_of(mine, own_units, a->max_len, 32);
    p.prefix_rt = std::max(p.own_rt, tiles_of(all, prefix_units, a->prefix_cap, bf16 ? 64 : 32));
    // Many: tiles of 128 queries, 64 where those times 128 rows are less than four a CU (400 queries of 8 heads behind 4096 rows 23.5 us and, with 64, 23.1, 512
    // behind 2048 20.5 and 18.3, behind 16384 59.6 and 71.2).
    if (p.form == SharedForm::many) p.prefix_rt = prefix_units * ceil_div(all, 128) * ceil_div(a->prefix_cap, 128) < 1024 ? 1 : 2;
    p.own_tiles = (int)ceil_div(mine, 16 * p.own_rt);
    p.prefix_tiles = (int)ceil_div(all, (p.form == SharedForm::many ? 64 : 16) * p.prefix_rt);
    p.prefix_parts = parts(prefix_units * p.prefix_tiles, 256, a->prefix_cap, bf16 || p.prefix_rt > 1 ? 128 : 64, kMostParts - 16);
    const long long others = std::min(256ll, prefix_units * p.prefix_tiles * p.prefix_parts);
    p.own_parts = parts(own_units * p.own_tiles, 512 - others, a->max_len, bf16 || p.own_rt > 1 ? 128 : 64, 16);
    p.prefix_blocks = ceil_div(prefix_units * p.prefix_parts, 8) * 8 * p.prefix_tiles;
    p.own_alone = p.own_parts == 1 && shared_alone(own_units * p.own_tiles, a->max_len, 256);
    p.own_blocks = p.own_alone ? ceil_div(own_units * p.own_tiles, 4) : ceil_div(own_units * p.own_parts, 8) * 8 * p.own_tiles;
  }
  const int all_parts = p.prefix_parts + p.own_parts;
  p.bytes = all_parts > 1 ? (size_t)all_parts * p.queries * (8 + 4 * (size_t)a->dim) : 0;
  return p;
}

SharedAttention shared_of(const ajqs_shared_attention_args* a, const SharedPlan& p, void* workspace) {
  SharedAttention s{};
  s.q = a->q;
  s.prefix_keys = a->prefix_keys;
  s.prefix_values = a->prefix_values;
  s.keys = a->keys;
  s.values = a->values;
  s.prefix_lengths = int64s(a->prefix_lengths);
  s.rows = int64s(a->rows);
  s.counts = int64s(a->counts);
  s.offset = int64s(a->offset);
  s.out = reinterpret_cast<uint16_t*>(a->out);
  s.part_sums = reinterpret_cast<float*>(workspace);
  s.part_ml = reinterpret_cast<float2*>(s.part_sums + (size_t)(p.prefix_parts + p.own_parts) * p.queries * a->dim);
  s.prefix_group = a->prefix_group;
  s.prefix_head = a->prefix_head;
  s.cache_batch = a->cache_batch;
  s.cache_head = a->cache_head;
  s.queries = p.queries;
  s.groups = a->groups;
  s.batch = a->batch;
  s.tokens = a->tokens;
  s.heads = a->heads;
  s.kv_heads = a->kv_heads;
  s.prefix_cap = a->prefix_cap;
  s.max_len = a->max_len;
  s.prefix_blocks = (int)p.prefix_blocks;
  s.prefix_parts = p.prefix_parts;
  s.prefix_tiles = p.prefix_tiles;
  s.own_parts = p.own_parts;
  s.own_tiles = p.own_tiles;
  s.own_alone = p.own_alone;
  s.scale2 = kLog2e / sqrtf((float)a->dim);
  s.by_share = divide_by(a->heads / a->kv_heads);
  s.by_each = divide_by((long long)a->tokens * (a->heads / a->kv_heads));
  s.by_tokens = divide_by(a->tokens);
  s.by_heads = divide_by(a->heads);
  s.by_kv_heads = divide_by(a->kv_heads);
  s.by_group = divide_by(a->batch / a->groups);
  s.by_prefix_tiles = divide_by(p.prefix_tiles);
  s.by_prefix_parts = divide_by(p.prefix_parts);
  s.by_own_tiles = divide_by(p.own_tiles);
  s.by_own_parts = divide_by(p.own_parts);
  return s;
}

template <int HD>
int merge_parts(const SharedAttention& s, const SharedPlan& p, hipStream_t stream, const char* what) {
  if (int e = check_launch(what)) return e;
  hipLaunchKernelGGL(shared_attention_merge_kernel<HD>, dim3((unsigned)ceil_div(p.queries, 4)), dim3(256), 0, stream, s);
  return check_launch(what);
}
template <int HD, typename QT, typename CacheT, int RTP, int RTO>
int launch_few(const SharedAttention& s, const SharedPlan& p, hipStream_t stream, const char* what) {
  constexpr int bytes = std::max(some_lds_bytes<HD, CacheT, RTP>(), some_lds_bytes<HD, CacheT, RTO>());
  auto kernel = shared_attention_few_kernel<HD, QT, CacheT, RTP, RTO>;
  if (int e = allow_lds(kernel, bytes, what)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(p.prefix_blocks + p.own_blocks)), dim3(256), bytes, stream, s);
  return merge_parts<HD>(s, p, stream, what);
}
template <int HD, typename QT, typename CacheT>
int launch_each(const SharedAttention& s, const SharedPlan& p, hipStream_t stream, const char* what) {
  constexpr int bytes = some_lds_bytes<HD, CacheT, 1>();
  auto kernel = shared_attention_each_kernel<HD, QT, CacheT>;
  if (int e = allow_lds(kernel, bytes, what)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.own_blocks), dim3(256), bytes, stream, s);
  return check_launch(what);
}
template <int HD, typename QT, int U>
int launch_many(const SharedAttention& s, const SharedPlan& p, hipStream_t stream, const char* what) {
  constexpr int bytes = std::max(many_lds_bytes<HD>(), few_lds_bytes<HD, uint16_t, 1>());
  auto kernel = shared_attention_many_kernel<HD, QT, U>;
  if (int e = allow_lds(kernel, bytes, what)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(p.prefix_blocks + p.own_blocks)), dim3(256), bytes, stream, s);
  return merge_parts<HD>(s, p, stream, what);
}
template <int HD, typename QT, int U>
int launch_walk(const SharedAttention& s, const SharedPlan& p, hipStream_t stream, const char* what) {
  auto kernel = shared_attention_walk_kernel<HD, QT, U>;
  if (int e = allow_lds(kernel, many_lds_bytes<HD>(), what)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.own_blocks), dim3(256), many_lds_bytes<HD>(), stream, s);
  return p.own_parts > 1 ? merge_parts<HD>(s, p, stream, what) : check_launch(what);
}

}  // namespace

extern "C" {

const char* ajqs_last_error(void) { return g_error; }

int ajqs_norm_rope(const ajqs_norm_rope_args* a, void* stream) { return ajqs_norm_rope_at(a, nullptr, 0, stream); }

int ajqs_norm_rope_at(const ajqs_norm_rope_args* a, const int64_t* depths, int64_t depths_ld, void* stream) {
  const char* what = "ajqs_norm_rope";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->qkv || !a->cosine || !a->sine || !a->rows || !a->keys || !a->values || !a->q)
    return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (!built_dim(a->dim)) return fail(AJQ_ERR_UNSUPPORTED, "%s: head size %d (128, 64 and 32 are built)", what, a->dim);
  if (a->batch < 1 || a->tokens < 1 || a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads != 0 || a->max_len < 1 || a->table_rows < 1 ||
      (long long)a->batch * a->tokens > 0x7FFFFFFFLL)
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (batch=%d tokens=%d heads=%d kv_heads=%d max_len=%d table_rows=%d)", what, a->batch,
                a->tokens, a->heads, a->kv_heads, a->max_len, a->table_rows);
  if ((long long)a->batch * a->tokens > kMostLanes / 256)
    return fail(AJQ_ERR_SHAPE, "%s: %d x %d tokens in a launch", what, a->batch, a->tokens);
  const long long all = (long long)a->heads + 2ll * a->kv_heads, room = (long long)a->max_len * a->dim;
  if (all > 1 << 20 || a->ld < all * a->dim || a->ld % 4 != 0)
    return fail(AJQ_ERR_SHAPE, "%s: rows of %lld elements (a multiple of 4, at least %lld)", what, (long long)a->ld, all * a->dim);
  if (!known(a->in_dtype) || !known(a->q_dtype) || !known(a->cache_dtype)) return fail(AJQ_ERR_UNSUPPORTED, "%s: unknown element type", what);
  if (!aligned16(a->qkv) || !aligned16(a->q) || !aligned16(a->cosine) || !aligned16(a->sine) || !aligned16(a->q_gain) || !aligned16(a->k_gain))
    return fail(AJQ_ERR_ALIGN, "%s: qkv, q, the tables and the gains must be 16-byte aligned", what);
  if (int e = check_caches(what, a->keys, a->values, a->cache_batch, a->cache_head)) return e;
  if (blocks_meet(0, a->cache_batch, a->batch, a->cache_head, a->kv_heads, room))
    return fail(AJQ_ERR_SHAPE, "%s: cache heads that overlap cannot be written", what);
  const int size = a->cache_dtype == AJQS_BF16 ? 2 : 4;
  const long long d = (long long)(reinterpret_cast<uintptr_t>(a->values) - reinterpret_cast<uintptr_t>(a->keys)) / size;
  if (d == 0 || blocks_meet(d, a->cache_batch, a->batch, a->cache_head, a->kv_heads, room))
    return fail(AJQ_ERR_SHAPE, "%s: keys and values that overlap cannot be written", what);
  if (depths && depths_ld < 0) return fail(AJQ_ERR_SHAPE, "%s: negative stride of the depths", what);
  if (!(a->eps >= 0.f)) return fail(AJQ_ERR_SHAPE, "%s: epsilon %g", what, a->eps);
  const NormRope n{a->qkv, a->cosine, a->sine, a->q_gain, a->k_gain, int64s(a->rows), int64s(a->positions), int64s(a->counts),
                   int64s(a->offset), int64s(depths), a->keys, a->values, a->q, a->ld, a->cache_batch, a->cache_head, depths_ld, a->tokens, a->heads, a->kv_heads,
                   a->max_len, a->table_rows, a->eps, divide_by(a->tokens)};
  with_dim(a->dim, [&](auto dim) {
    with_type(a->in_dtype, [&](auto in) {
      with_type(a->q_dtype, [&](auto q) {
        with_type(a->cache_dtype, [&](auto cache) {
          auto launch = [&](auto each, auto many) {
            constexpr int U = decltype(each)::value;
            const dim3 grid((unsigned)(a->batch * a->tokens), (unsigned)ceil_div(all, 16 * U));
            hipLaunchKernelGGL((norm_rope_kernel<decltype(in), decltype(q), decltype(cache), decltype(dim)::value, U, decltype(many)::value>), grid,
                               dim3(256), 0, (hipStream_t)stream, n);
          };
          const std::integral_constant<bool, true> yes;
          const std::integral_constant<bool, false> no;
          // one head a team until there are workgroups enough, then two or three, whichever leaves fewer of a token's teams idle (16 prompts of 333 tokens, one, two and
          // three: 48 heads 33.3, 31.2 and 28.5 us, 96 63.6, 52.5 and 50.5, 32 23.9, 20.9 and 21.4, 36 of 64 18.3, 17.0 and 14.6; 2 of 333, 48 6.7, 6.6 and 6.8)
          const bool full = (long long)a->batch * a->tokens >= 1024;
          if (a->tokens == 1) full && all > 16 ? launch(Size<2>{}, no) : launch(Size<1>{}, no);
          else if (!full || all <= 16) launch(Size<1>{}, yes);
          else ceil_div(all, 48) * 48 > ceil_div(all, 32) * 32 ? launch(Size<2>{}, yes) : launch(Size<3>{}, yes);
        });
      });
    });
  });
  return check_launch(what);
}

size_t ajqs_shared_attention_workspace(const ajqs_shared_attention_args* a) { return check_shared(a) ? 0 : shared_plan(a).bytes; }

int ajqs_shared_attention(const ajqs_shared_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "ajqs_shared_attention";
  if (int e = check_shared(a)) return e;
  const SharedPlan p = shared_plan(a);
  if (p.prefix_blocks + p.own_blocks > kMostLanes / 256) return fail(AJQ_ERR_SHAPE, "%s: too many tiles of queries", what);
  if (p.bytes && ceil_div(p.queries, 4) > kMostLanes / 256) return fail(AJQ_ERR_SHAPE, "%s: too many queries (%lld)", what, p.queries);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes))
    return fail(AJQ_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, p.bytes, workspace_bytes);
  if (!aligned16(workspace)) return fail(AJQ_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", what);
  const SharedAttention s = shared_of(a, p, workspace);
  int status = AJQ_OK;
  with_dim(a->dim, [&](auto dim) {
    with_type(a->q_dtype, [&](auto q) {
      with_type(a->cache_dtype, [&](auto cache) {
        constexpr int HD = decltype(dim)::value;
        using QT = decltype(q);
        using CacheT = decltype(cache);
        if constexpr (sizeof(CacheT) == 2) {
          if (p.form == SharedForm::walk) {
            if constexpr (HD == 128 && sizeof(QT) == 2) {
              if (p.own_rt == 2) {
                status = launch_walk<HD, QT, 2>(s, p, (hipStream_t)stream, what);
                return;
              }
            }
            status = launch_walk<HD, QT, 1>(s, p, (hipStream_t)stream, what);
            return;
          }
          if (p.form == SharedForm::many) {
            status = p.prefix_rt == 2 ? launch_many<HD, QT, 2>(s, p, (hipStream_t)stream, what) : launch_many<HD, QT, 1>(s, p, (hipStream_t)stream, what);
            return;
          }
        }
        if (p.form == SharedForm::each) {
          status = launch_each<HD, QT, CacheT>(s, p, (hipStream_t)stream, what);
          return;
        }
        if constexpr (sizeof(CacheT) == 4) {
          if (p.own_rt == 2) {
            status = launch_few<HD, QT, CacheT, 2, 2>(s, p, (hipStream_t)stream, what);
            return;
          }
        }
        const auto launch = p.prefix_rt == 2 ? launch_few<HD, QT, CacheT, 2, 1> : launch_few<HD, QT, CacheT, 1, 1>;
        status = launch(s, p, (hipStream_t)stream, what);
      });
    });
  });
  return status;
}

int ajqs_adjust_logits(const ajqs_adjust_logits_args* a, void* stream) {
  const char* what = "ajqs_adjust_logits";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->logits || !a->out || (a->bias_ids && !a->bias)) return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (a->batch < 1 || a->vocab < 1 || a->ld < a->vocab || a->out_ld < a->vocab)
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (batch=%d vocab=%d ld=%lld out_ld=%lld)", what, a->batch, a->vocab, (long long)a->ld,
                (long long)a->out_ld);
  if (!known(a->dtype)) return fail(AJQ_ERR_UNSUPPORTED, "%s: unknown element type", what);
  if (a->logits == a->out && (a->dtype != AJQS_F32 || a->ld != a->out_ld))
    return fail(AJQ_ERR_UNSUPPORTED, "%s: only fp32 logits can be adjusted in place, row by row", what);
  // (read only: a stride of 0 is one list, or mask, for all rows)
  auto rows_of = [](long long stride, long long width) { return stride == 0 || stride >= width; };
  if (a->tokens && (a->max_tokens < 0 || a->max_tokens > kMaxHistory || !rows_of(a->tokens_ld, a->max_tokens)))
    return fail(AJQ_ERR_SHAPE, "%s: %d tokens a row (at most %d, and the rows' stride %lld)", what, a->max_tokens, kMaxHistory,
                (long long)a->tokens_ld);
  if (a->prompt && (a->max_prompt < 0 || a->max_prompt > kMaxHistory || !rows_of(a->prompt_ld, a->max_prompt)))
    return fail(AJQ_ERR_SHAPE, "%s: %d prompt tokens a row (at most %d, and the rows' stride %lld)", what, a->max_prompt, kMaxHistory,
                (long long)a->prompt_ld);
  if (a->bias_ids && (a->biases < 0 || a->biases > kMaxBiases || a->bias_ld < a->biases))
    return fail(AJQ_ERR_SHAPE, "%s: %d biases a row (at most %d, and the rows' stride %lld)", what, a->biases, kMaxBiases, (long long)a->bias_ld);
  if (a->allowed && (a->masks < 1 || !rows_of(a->allowed_ld, ((long long)a->vocab + 31) / 32)))
    return fail(AJQ_ERR_SHAPE, "%s: masks of %lld words for a vocabulary of %d", what, (long long)a->allowed_ld, a->vocab);
  if (a->allowed && !a->allowed_rows && a->masks < a->batch)
    return fail(AJQ_ERR_SHAPE, "%s: %d masks for %d rows", what, a->masks, a->batch);
  if (!aligned4(a->out) || !aligned4(a->allowed) || (a->dtype == AJQS_F32 && !aligned4(a->logits)) || (reinterpret_cast<uintptr_t>(a->logits) & 1u))
    return fail(AJQ_ERR_ALIGN, "%s: logits, out and the masks must be aligned to their elements", what);
  const int size = a->dtype == AJQS_BF16 ? 2 : 4;
  if (a->logits != a->out && rows_meet(a->logits, a->ld * size, (long long)a->vocab * size, a->out, a->out_ld * 4, (long long)a->vocab * 4, a->batch))
    return fail(AJQ_ERR_SHAPE, "%s: out overlaps the logits without being them", what);
  const bool words = (a->tokens && a->max_tokens) || (a->prompt && a->max_prompt) || (a->bias_ids && a->biases);
  // Slices of 16384 tokens (two workgroups of 1024 lanes a CU then; 256 rows of 128256 66 us, 75 in slices of 8192, whose rows' lists are read twice as often),
  // smaller ones until there are two workgroups a CU (8 rows 6.2 us, 8.2 with one a CU, 6.4 with four; 64 rows 15.7, 16.0 and 20.0).
  int slice = 4 * kSliceThreads * kSlicePieces;
  while (slice > 1024 && (long long)a->batch * ceil_div(a->vocab, slice) < 512) slice /= 2;
  const int threads = std::min(slice / 4, std::max(256, slice / (4 * kSlicePieces))), slices = (int)ceil_div(a->vocab, slice);
  const long long blocks = ceil_div(a->batch, 8) * 8 * slices;
  if (blocks > kMostLanes / threads) return fail(AJQ_ERR_SHAPE, "%s: %d rows of %d", what, a->batch, a->vocab);
  const AdjustLogits n{a->logits, a->out, a->max_tokens ? int64s(a->tokens) : nullptr, int64s(a->token_counts), a->max_prompt ? int64s(a->prompt) : nullptr, int64s(a->prompt_counts),
                       a->repetition, a->frequency, a->presence, int64s(a->bias_ids), a->bias, a->allowed, int64s(a->allowed_rows), a->ld, a->out_ld, a->tokens_ld,
                       a->prompt_ld, a->bias_ld, a->allowed_ld, a->vocab, a->max_tokens, a->max_prompt, a->bias_ids ? a->biases : 0, a->masks,
                       a->token_count_stride, a->prompt_count_stride, a->batch, slice, slices};
  int status = AJQ_OK;
  with_type(a->dtype, [&](auto type) {
    using T = decltype(type);
    auto launch = [&](auto with_words, auto in_place) {
      auto kernel = adjust_logits_kernel<T, decltype(with_words)::value, decltype(in_place)::value>;
      const int bytes = decltype(with_words)::value ? slice * 4 : 0;
      if ((status = allow_lds(kernel, bytes, what)) == AJQ_OK)
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), bytes, (hipStream_t)stream, n);
    };
    const std::integral_constant<bool, true> yes;
    const std::integral_constant<bool, false> no;
    auto for_words = [&](auto in_place) { words ? launch(yes, in_place) : launch(no, in_place); };
    if constexpr (sizeof(T) == 4) {
      if (a->logits == a->out) return for_words(yes);
    }
    for_words(no);
  });
  if (status) return status;
  return check_launch(what);
}

}  // extern "C"
