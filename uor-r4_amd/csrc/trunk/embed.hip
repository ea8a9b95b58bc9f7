// embed.hip - the lookup of tokens' rows, scaled, and its gradient by sorted tokens:
//
//   y_t = scale E[token_t],   dE_v = scale sum of dy_t over the rows t whose token is v.
//
// Both are bound by the rows' bytes.
#include "sorted.h"

namespace trunk {

struct Embed {
  uint32_t rows, vocab, width;
  bool wide;
  float scale;
  int64_t table_stride;
  const void *tokens, *table;
  void *y;
};

// LANES lanes take a row, eight values at a time; four rows at a time, so that their tokens and then their
// rows are on their way together.
template <class E, class T, int LANES>
__global__ __launch_bounds__(256) void embed_rows(Embed a) {
  constexpr uint32_t kRows = 256 / LANES, kAhead = 4;
  const uint32_t lane = threadIdx.x % LANES;
  for (uint64_t base = (uint64_t)blockIdx.x * kRows * kAhead + threadIdx.x / LANES; base < a.rows; base += (uint64_t)gridDim.x * kRows * kAhead) {
    uint32_t token[kAhead];
#pragma unroll
    for (uint32_t k = 0; k < kAhead; k++) {
      const uint64_t row = base + k * kRows;
      token[k] = row < a.rows ? token_of(a.tokens, a.wide, row, a.vocab) : a.vocab;
    }
    for (uint32_t eight = lane; eight * 8 < a.width; eight += LANES) {
      const uint32_t col = eight_of(eight, a.width);
      f32x8 v[kAhead];
#pragma unroll
      for (uint32_t k = 0; k < kAhead; k++)
        v[k] = __builtin_convertvector((load_some<E, 8>((const E *)a.table + (int64_t)token[k] * a.table_stride, token[k] < a.vocab, col, a.width)), f32x8);
#pragma unroll
      for (uint32_t k = 0; k < kAhead; k++) {
        const uint64_t row = base + k * kRows;
        if (row >= a.rows) break;
        v[k] = token[k] < a.vocab ? v[k] * a.scale : f32x8{};
        // In bf16 past the caches, which hold the table meanwhile: 262,144 rows of 256 33.6 us, through them 36.4; 131,072 of 512 from
        // 131,072 words 29.8 and 35.5.
        store_past<T>((T *)a.y + row * a.width, col, a.width, __builtin_convertvector(v[k], V8<T>));
      }
    }
  }
}

namespace {

int check_embed(const uor_trunk_embed_args *s) {
  if (!s) return fail(-1, "null argument");
  if (s->dtype > UOR_TRUNK_F32 || s->table_dtype > UOR_TRUNK_F32) return fail(-1, "dtype %u or %u is neither bf16 nor f32", s->dtype, s->table_dtype);
  if (s->width < 1 || s->width > UOR_TRUNK_MAX_WIDTH) return fail(-1, "width %u outside 1..8192", s->width);
  if (s->vocab < 1 || s->vocab > UOR_TRUNK_MAX_VOCAB) return fail(-1, "a vocabulary of %u outside 1..%u", s->vocab, UOR_TRUNK_MAX_VOCAB);
  if (s->rows > UOR_TRUNK_MAX_ROWS) return fail(-1, "%u rows are more than %u", s->rows, UOR_TRUNK_MAX_ROWS);
  if (s->rows && !s->tokens) return fail(-1, "null tokens");
  return 0;
}
template <class E, class T>
int look_up(const Embed &a, hipStream_t stream) {
  with_lanes(a.width, [&](auto lanes) {
    constexpr uint32_t kRows = 256 / lanes() * 4;
    const uint32_t blocks = (a.rows + kRows - 1) / kRows;
    hipLaunchKernelGGL((embed_rows<E, T, lanes()>), dim3(blocks < 8192 ? blocks : 8192), dim3(256), 0, stream, a);
  });
  return launched();
}

}  // namespace
}  // namespace trunk

using namespace trunk;

extern "C" uint64_t uor_trunk_sizeof_embed(void) { return sizeof(uor_trunk_embed_args); }

extern "C" int uor_trunk_embed_async(const uor_trunk_embed_args *s, void *stream) {
  if (const int e = check_embed(s)) return e;
  if (!s->rows) return 0;
  if (!s->table || !s->y) return fail(-1, "null table or y");
  if (s->vocab > 1 && s->table_stride < s->width) return fail(-1, "the table's rows overlap: a stride is less than a row");
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  const Embed a{s->rows, s->vocab, s->width, s->wide != 0, s->scale, s->table_stride, s->tokens, s->table, s->y};
  const bool half = s->dtype == UOR_TRUNK_BF16;
  if (s->table_dtype == UOR_TRUNK_BF16) return half ? look_up<bf16, bf16>(a, (hipStream_t)stream) : look_up<bf16, float>(a, (hipStream_t)stream);
  return half ? look_up<float, bf16>(a, (hipStream_t)stream) : look_up<float, float>(a, (hipStream_t)stream);
}

extern "C" uint64_t uor_trunk_embed_backward_workspace_bytes(const uor_trunk_embed_args *s) {
  return check_embed(s) ? 0 : sort_plan(s->rows, s->vocab, s->width).bytes;
}

extern "C" int uor_trunk_embed_backward_async(const uor_trunk_embed_args *s, void *workspace, uint64_t bytes, void *stream) {
  if (const int e = check_embed(s)) return e;
  if (!s->dtable || (s->rows && !s->dy)) return fail(-1, "null dy or dtable");
  if (s->rows > 1 && s->dy_stride < s->width) return fail(-1, "rows overlap: a stride is less than a row");
  const SortPlan p = sort_plan(s->rows, s->vocab, s->width);
  if (p.bytes && (!workspace || bytes < p.bytes || (uintptr_t)workspace % 16))
    return fail(-1, "a workspace of %llu bytes, aligned to 16, is wanted", (unsigned long long)p.bytes);
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  const hipStream_t on_stream = (hipStream_t)stream;
  Sums a{};
  a.width = s->width, a.words = s->vocab, a.scale = s->scale;
  a.stride = s->dy_stride, a.pitch = s->width, a.from = s->dy, a.to = s->dtable;
  sort_rows(p, s->tokens, s->wide != 0, s->rows, s->vocab, (char *)workspace, on_stream, a);
  const bool half = s->dtype == UOR_TRUNK_BF16;
  if (s->table_dtype == UOR_TRUNK_BF16) half ? sum_rows<bf16, bf16>(a, on_stream) : sum_rows<bf16, float>(a, on_stream);
  else half ? sum_rows<float, bf16>(a, on_stream) : sum_rows<float, float>(a, on_stream);
  return launched();
}
