// The OpEnvs of the operators at the vocabulary against a recording stand-in for the kernel library,
// driven through the C window: a descriptor that differs from the one the OpEnv was made with in
// shape, dtype or device is refused before anything reaches the library.  No GPU, no HIP.
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "rafhip_dialect.h"
#include "rafhip_vocab.h"

#define EXPECT(cond)                                                \
  do {                                                              \
    if (!(cond)) {                                                  \
      std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      return 1;                                                     \
    }                                                               \
  } while (0)

// ------------------------------------------------------------- the recording kernel library
static int g_calls = 0;
static int32_t g_index_bits = 0;
static int64_t g_tokens = 0;

extern "C" {
int rafhip_device_count(void) { return 1; }
const char* rafhip_last_error(void) { return "recording stand-in"; }
int rafhip_embedding(const void*, int32_t, int64_t, int64_t, const void*, int32_t index_bits, int64_t n, int64_t, float, void*,
                     int32_t, void*) {
  ++g_calls;
  g_index_bits = index_bits;
  g_tokens = n;
  return RAFHIP_OK;
}
int64_t rafhip_embedding_dx_workspace_bytes(int64_t, int64_t, int64_t) { return 64; }
int rafhip_embedding_dx(const void*, int32_t, const void*, int32_t index_bits, int64_t n, int64_t, int64_t, int64_t, int32_t,
                        int64_t, float, void*, int32_t, int32_t, void*, int64_t, void*) {
  ++g_calls;
  g_index_bits = index_bits;
  g_tokens = n;
  return RAFHIP_OK;
}
int64_t rafhip_topk_distill_workspace_bytes(const rafhip_topk_distill_args*) { return 64; }
int rafhip_topk_distill(const rafhip_topk_distill_args*, float*, float*, void*, int64_t, void*) {
  ++g_calls;
  return RAFHIP_OK;
}
int rafhip_topk_distill_dx(const rafhip_topk_distill_args*, const float*, int64_t, const float*, void*, int64_t, void*) {
  ++g_calls;
  return RAFHIP_OK;
}
int rafhip_topk_distill_step(const rafhip_topk_distill_args*, const float*, int64_t, float*, void*, int64_t, void*, int64_t,
                             void*) {
  ++g_calls;
  return RAFHIP_OK;
}
}  // extern "C"

static char g_memory[4096];
static const int32_t kRocm = 10;
static const int32_t kInt = 0, kFloat = 2, kBfloat = 4;

struct Desc {
  rafhip_tensor_desc d;
  std::vector<int64_t> shape;
  Desc(int32_t code, int32_t bits, std::vector<int64_t> s, void* data = g_memory) : shape(std::move(s)) {
    d = rafhip_tensor_desc{data, kRocm, 0, code, bits, (int32_t)shape.size(), nullptr};
  }
  const rafhip_tensor_desc* get() {
    d.shape = shape.data();
    return &d;
  }
};

static rafhip_tensor_desc Absent() { return rafhip_tensor_desc{nullptr, 0, 0, 0, 0, -1, nullptr}; }

static char g_workspace[4096];

static int Run(rafhip_raf_env* env, const std::vector<rafhip_tensor_desc>& in, const std::vector<rafhip_tensor_desc>& out) {
  return rafhip_raf_execute(env, (int32_t)in.size(), in.data(), (int32_t)out.size(), out.data(), g_workspace,
                            sizeof(g_workspace), nullptr);
}

static bool Says(const char* text) { return std::strstr(rafhip_raf_last_error(), text) != nullptr; }

// Every tensor of a call in turn with another shape, dtype (of more and of fewer bits) and device:
// all refused, none reaches the library; then the call itself, which does.
static int TryAll(const char* op, rafhip_raf_env* env, const std::vector<rafhip_tensor_desc>& in,
                  const std::vector<rafhip_tensor_desc>& out) {
  std::puts(op);
  const size_t n = in.size() + out.size();
  for (size_t at = 0; at < n; ++at) {
    auto with = [&](auto change) {
      std::vector<rafhip_tensor_desc> i = in, o = out;
      rafhip_tensor_desc& d = at < in.size() ? i[at] : o[at - in.size()];
      change(d);
      return Run(env, i, o);
    };
    if ((at < in.size() ? in[at] : out[at - in.size()]).ndim < 0) continue;
    const int before = g_calls;
    for (int32_t bits : {8, 16, 32, 64}) {
      if (bits == (at < in.size() ? in[at] : out[at - in.size()]).dtype_bits) continue;
      EXPECT(with([&](rafhip_tensor_desc& d) { d.dtype_bits = bits; }) != 0 && Says("dtype"));
    }
    EXPECT(with([&](rafhip_tensor_desc& d) { d.dtype_code = d.dtype_code == kFloat ? kBfloat : kFloat; }) != 0 && Says("dtype"));
    EXPECT(with([&](rafhip_tensor_desc& d) { d.device_id = 1; }) != 0 && Says("device"));
    EXPECT(with([&](rafhip_tensor_desc& d) { d.device_type = 1; }) != 0 && Says("device"));
    EXPECT(with([&](rafhip_tensor_desc& d) {
             static const int64_t other[] = {1, 2, 3, 4, 5, 6, 7};
             d.shape = other;
             d.ndim = 7;
           }) != 0 && Says("shape"));
    EXPECT(with([&](rafhip_tensor_desc& d) { d.ndim = -1; }) != 0);  // missing
    EXPECT(g_calls == before);
  }
  const int before = g_calls;
  EXPECT(Run(env, in, out) == 0);
  EXPECT(g_calls == before + 1);
  EXPECT(Run(env, std::vector<rafhip_tensor_desc>(in.begin(), in.end() - 1), out) != 0);
  std::vector<rafhip_tensor_desc> more = out;
  more.push_back(out[0]);
  EXPECT(Run(env, in, more) != 0);
  EXPECT(g_calls == before + 1);
  return 0;
}

int main() {
  rafhip_raf_env* env = nullptr;
  for (int32_t bits : {32, 64}) {
    Desc x(kFloat, 32, {6, 4}), ids(kInt, bits, {5}), y(kBfloat, 16, {5, 4});
    EXPECT(rafhip_raf_embedding_make(x.get(), ids.get(), 2.0, 0, kBfloat, 16, &env) == 0);
    if (TryAll("embedding", env, {*x.get(), *ids.get()}, {*y.get()})) return 1;
    EXPECT(g_index_bits == bits && g_tokens == 5);
    rafhip_raf_env_destroy(env);

    Desc dy(kBfloat, 16, {5, 4}), dx(kFloat, 32, {6, 4}, g_memory + 1024);
    EXPECT(rafhip_raf_embedding_dx_make(dy.get(), ids.get(), nullptr, 6, 1.0, 0, 0, 0, kFloat, 32, &env) == 0);
    if (TryAll("embedding_dx", env, {*dy.get(), *ids.get(), Absent()}, {*dx.get()})) return 1;
    EXPECT(g_index_bits == bits && g_tokens == 5);
    EXPECT(Run(env, {*dy.get(), *ids.get(), *dx.get()}, {*dx.get()}) != 0 && Says("grad came or went"));
    rafhip_raf_env_destroy(env);
    EXPECT(rafhip_raf_embedding_dx_make(dy.get(), ids.get(), dx.get(), 6, 1.0, 0, 0, 0, kFloat, 32, &env) == 0);
    if (TryAll("embedding_dx into grad", env, {*dy.get(), *ids.get(), *dx.get()}, {*dx.get()})) return 1;
    Desc elsewhere(kFloat, 32, {6, 4}, g_memory + 2048);
    EXPECT(Run(env, {*dy.get(), *ids.get(), *dx.get()}, {*elsewhere.get()}) != 0 && Says("is grad"));
    rafhip_raf_env_destroy(env);
  }
  Desc z(kFloat, 16, {3, 9}), index(kInt, 32, {3, 2}), top(kFloat, 32, {3, 2}), labels(kInt, 32, {3}), dloss(kFloat, 32, {3}),
      stats(kFloat, 32, {3, 3}), loss(kFloat, 32, {3}), dz(kFloat, 16, {3, 9});
  for (bool labelled : {false, true}) {
    const rafhip_tensor_desc* l = labelled ? labels.get() : nullptr;
    const rafhip_tensor_desc given = labelled ? *l : Absent();
    EXPECT(rafhip_raf_topk_distill_make(0, z.get(), index.get(), top.get(), l, nullptr, nullptr, 2.0, 1.0, 0.5, 9, &env) == 0);
    if (TryAll("topk_distill", env, {*z.get(), *index.get(), *top.get(), given, Absent(), Absent()}, {*loss.get(), *stats.get()}))
      return 1;
    rafhip_raf_env_destroy(env);
    EXPECT(rafhip_raf_topk_distill_make(1, z.get(), index.get(), top.get(), l, dloss.get(), stats.get(), 2.0, 1.0, 0.5, 9, &env) ==
           0);
    if (TryAll("topk_distill_dx", env, {*z.get(), *index.get(), *top.get(), given, *dloss.get(), *stats.get()}, {*dz.get()}))
      return 1;
    rafhip_raf_env_destroy(env);
    EXPECT(rafhip_raf_topk_distill_make(2, z.get(), index.get(), top.get(), l, dloss.get(), nullptr, 2.0, 1.0, 0.5, 9, &env) == 0);
    if (TryAll("topk_distill_step", env, {*z.get(), *index.get(), *top.get(), given, *dloss.get(), Absent()},
               {*loss.get(), *dz.get()}))
      return 1;
    rafhip_raf_env_destroy(env);
  }
  std::puts("ALL OK");
  return 0;
}
