// Host checks of the quantised KV cache: the tile layout of kv_quant.cuh, and
// the refusals of the C entry points that need no device.  Prints "ok" or the
// first failure.
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "../include/uocr_q8.h"
#include "../unlimited-ocr-kernel_b200/csrc/handles.h"

using namespace uocr;

static int fail(const char* what, int a = 0, int b = 0, int c = 0) {
  std::printf("%s (%d, %d, %d)\n", what, a, b, c);
  return 1;
}

// Every (token, dim) has a nibble (or byte) of its own, no byte is shared by
// two tokens, the parameters have words of their own, and all lie in the tile.
static int layout() {
  for (int bits : {4, 8})
    for (int dim = 1; dim <= kKvqMaxDim; ++dim) {
      const KvqLayout L = kvq_layout(3, dim, bits, 33);
      if (L.tiles != 2 || L.groups != (dim + 31) / 32) return fail("counts", bits, dim);
      if (L.codes != L.groups * 32 * 32 * bits / 8 || L.half % 16 || L.tile != 2 * L.half)
        return fail("sizes", bits, dim);
      for (int value = 0; value < 2; ++value) {
        std::vector<int> nibbles(2 * L.codes, 0), owner(L.codes, -1);
        for (int t = 0; t < 32; ++t)
          for (int d = 0; d < L.groups * 32; ++d) {
            const int at = value ? kvq_value_byte(t, d, bits) : kvq_key_byte(t, d, bits);
            const int nib = bits == 8 ? 0 : value ? kvq_value_nibble(d) : kvq_key_nibble(d);
            if (at < 0 || at >= L.codes) return fail("code out of the tile", bits, t, d);
            if (owner[at] >= 0 && owner[at] != t) return fail("a byte of two tokens", bits, t, d);
            owner[at] = t;
            if (nibbles[2 * at + nib]++) return fail("a code of two dims", bits, t, d);
          }
        for (int at = 0; at < L.codes; ++at)
          if (owner[at] < 0) return fail("an unused byte", bits, dim, at);
      }
      std::vector<int> words(L.groups * 32, 0);
      for (int t = 0; t < 32; ++t)
        for (int g = 0; g < L.groups; ++g) {
          const int at = kvq_param_byte(t, g);
          if (at % 4 || at < 0 || at >= L.groups * 128 || words[at / 4]++)
            return fail("parameter word", bits, t, g);
        }
    }
  return 0;
}

#define EXPECT(call, code)                                                                   \
  do {                                                                                       \
    const int got = (call);                                                                  \
    if (got != (code)) {                                                                     \
      std::printf("%s: %d (%s), expected %d\n", #call, got, uocr_last_error(), (code));      \
      return 1;                                                                              \
    }                                                                                        \
  } while (0)

static int refusals() {
  uocr_ctx ctx;
  ctx.scratch_limit = 1 << 20;
  uocr_kvq* out = nullptr;
  EXPECT(uocr_kvq_create(nullptr, 1, 1, 32, 1, 1, 4, &out), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_create(&ctx, 1, 1, 32, 1, 1, 4, nullptr), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_create(&ctx, 1, 0, 32, 1, 1, 4, &out), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_create(&ctx, 1, 1, 0, 1, 1, 4, &out), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_create(&ctx, 1, 1, 32, 0, 1, 4, &out), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_create(&ctx, 0, 1, 32, 1, 1, 4, &out), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_create(&ctx, 1, 1, 32, 1, 0, 4, &out), UOCR_ERR_SHAPE);
  for (int bits : {-4, 0, 2, 5, 16, 32})
    EXPECT(uocr_kvq_create(&ctx, 1, 1, 32, 1, 1, bits, &out), UOCR_ERR_UNSUPPORTED);
  EXPECT(uocr_kvq_create(&ctx, 1, 1, 257, 1, 1, 4, &out), UOCR_ERR_UNSUPPORTED);
  EXPECT(uocr_kvq_create(&ctx, 1, 65536, 32, 1, 1, 4, &out), UOCR_ERR_UNSUPPORTED);
  EXPECT(uocr_kvq_create(&ctx, 65536, 1, 32, 1, 1, 4, &out), UOCR_ERR_UNSUPPORTED);
  EXPECT(uocr_kvq_create(&ctx, 1, 1, 32, 1, (size_t(1) << 30), 4, &out), UOCR_ERR_RESOURCE);
  EXPECT(uocr_kvq_create(&ctx, 1, 1, 32, SIZE_MAX, 2, 4, &out), UOCR_ERR_RESOURCE);
  EXPECT(uocr_kvq_create(&ctx, 1, SIZE_MAX, 3, 1, 1, 4, &out), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_create(&ctx, 65535, 65535, 256, 1, 1 << 29, 8, &out), UOCR_ERR_RESOURCE);

  uocr_kvq kv;
  kv.batch = 2;
  kv.width = 64;
  kv.window = 4;
  kv.max_prefix = 40;
  kv.layout = kvq_layout(2, 32, 4, 44);
  kv.prefix.assign(2, 0);
  float* p = reinterpret_cast<float*>(16);  // never read: every call below is refused
  EXPECT(uocr_kvq_prefill(nullptr, &kv, 0, p, 0, p, 0, 1), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_prefill(&ctx, nullptr, 0, p, 0, p, 0, 1), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_prefill(&ctx, &kv, 2, p, 0, p, 0, 1), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_prefill(&ctx, &kv, 0, p, 0, p, 0, 0), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_prefill(&ctx, &kv, 0, p, 0, p, 0, 41), UOCR_ERR_RESOURCE);
  EXPECT(uocr_kvq_prefill(&ctx, &kv, 0, nullptr, 0, p, 0, 1), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_prefill(&ctx, &kv, 0, p, 0, nullptr, 0, 1), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_prefill(&ctx, &kv, 0, p, 63, p, 0, 1), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_prefill(&ctx, &kv, 0, p, 0, p, SIZE_MAX, 1), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_push(&ctx, &kv, p, 0, p, 0), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_attention(&ctx, &kv, p, p), UOCR_ERR_SHAPE);
  kv.prefix[0] = 3;  // the other sequence is still empty
  EXPECT(uocr_kvq_prefill(&ctx, &kv, 0, p, 0, p, 0, 1), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_push(&ctx, &kv, p, 0, p, 0), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_attention(&ctx, &kv, p, p), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_read(&ctx, &kv, 1, 0, 1, p, p), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_read(&ctx, &kv, 2, 0, 1, p, p), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_read(&ctx, &kv, 0, 0, 8, p, p), UOCR_ERR_SHAPE);  // 3 + window
  EXPECT(uocr_kvq_read(&ctx, &kv, 0, 8, 0, p, p), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_read(&ctx, &kv, 0, 2, SIZE_MAX, p, p), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_read(&ctx, &kv, 0, 1, 1, nullptr, p), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_read(&ctx, &kv, 0, 7, 0, nullptr, nullptr), UOCR_OK);
  kv.prefix[1] = 1;
  EXPECT(uocr_kvq_push(&ctx, &kv, nullptr, 0, p, 0), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_push(&ctx, &kv, p, 1, p, 0), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_attention(&ctx, &kv, nullptr, p), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_attention(&ctx, &kv, p, nullptr), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_reset(&ctx, &kv, 2), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_state(&ctx, &kv, 2, nullptr, nullptr), UOCR_ERR_SHAPE);
  uocr_rope rope;
  rope.head_dim = 64;
  EXPECT(uocr_kvq_rope(&ctx, &kv, nullptr, p, p), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_rope(&ctx, &kv, &rope, p, p), UOCR_ERR_SHAPE);
  EXPECT(uocr_kvq_rope_push_qkv(&ctx, &kv, &rope, p, p), UOCR_ERR_SHAPE);
  rope.head_dim = 32;
  rope.device = 1;
  EXPECT(uocr_kvq_rope_push_qkv(&ctx, &kv, &rope, p, p), UOCR_ERR_INVALID);
  kv.device = 1;  // a cache of another device than the context's
  EXPECT(uocr_kvq_push(&ctx, &kv, p, 0, p, 0), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_read(&ctx, &kv, 0, 0, 1, p, p), UOCR_ERR_INVALID);
  EXPECT(uocr_kvq_free(nullptr), UOCR_OK);
  if (uocr_kvq_storage_bytes(nullptr) != 0) return fail("storage bytes of no cache");

  const int64_t* t = reinterpret_cast<const int64_t*>(16);
  int64_t* ids = reinterpret_cast<int64_t*>(16);
  EXPECT(uocr_token_logprobs(nullptr, p, 1, 8, 0, t, 0, p, p, nullptr, nullptr), UOCR_ERR_INVALID);
  EXPECT(uocr_token_logprobs(&ctx, p, 1, 0, 0, t, 0, p, p, nullptr, nullptr), UOCR_ERR_SHAPE);
  EXPECT(uocr_token_logprobs(&ctx, p, 1, 8, 7, t, 0, p, p, nullptr, nullptr), UOCR_ERR_SHAPE);
  EXPECT(uocr_token_logprobs(&ctx, p, 1, 8, 0, t, 9, p, p, ids, p), UOCR_ERR_SHAPE);
  EXPECT(uocr_token_logprobs(&ctx, p, 1, 64, 0, t, 33, p, p, ids, p), UOCR_ERR_UNSUPPORTED);
  EXPECT(uocr_token_logprobs(&ctx, p, 1, (size_t(1) << 30) + 1, 0, t, 0, p, p, nullptr, nullptr),
         UOCR_ERR_UNSUPPORTED);
  EXPECT(uocr_token_logprobs(&ctx, p, size_t(1) << 31, 8, 0, t, 0, p, p, nullptr, nullptr),
         UOCR_ERR_UNSUPPORTED);
  EXPECT(uocr_token_logprobs(&ctx, nullptr, 1, 8, 0, t, 0, p, p, nullptr, nullptr), UOCR_ERR_INVALID);
  EXPECT(uocr_token_logprobs(&ctx, p, 1, 8, 0, t, 0, nullptr, p, nullptr, nullptr), UOCR_ERR_INVALID);
  EXPECT(uocr_token_logprobs(&ctx, p, 1, 8, 0, nullptr, 0, p, p, nullptr, nullptr), UOCR_ERR_INVALID);
  EXPECT(uocr_token_logprobs(&ctx, p, 1, 8, 0, t, 2, p, p, nullptr, p), UOCR_ERR_INVALID);
  EXPECT(uocr_token_logprobs(&ctx, p, 1, 8, 0, t, 2, p, p, ids, nullptr), UOCR_ERR_INVALID);
  EXPECT(uocr_token_logprobs(&ctx, nullptr, 0, 8, 0, nullptr, 0, nullptr, nullptr, nullptr, nullptr),
         UOCR_OK);
  return 0;
}

int main(int argc, char** argv) {
  const std::string which = argc > 1 ? argv[1] : "";
  const int rc = which == "layout" ? layout() : which == "refusals" ? refusals() : fail("usage");
  if (!rc) std::puts("ok");
  return rc;
}
