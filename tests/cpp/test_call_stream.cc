// The device API's stream: SetStream holds for the process, whichever thread executes, and a call of
// the C window runs on the stream it names, whatever other threads set or run meanwhile.  The kernel
// library is a stand-in whose SGD step and lookup note the stream they are given.
#include <atomic>
#include <cstdio>
#include <thread>
#include <vector>

#include "raf_iface.h"
#include "rafhip_dialect.h"
#include "rafhip_vocab.h"

using namespace raf;
using namespace raf::op;

#define EXPECT(cond)                                                \
  do {                                                              \
    if (!(cond)) {                                                  \
      std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      return 1;                                                     \
    }                                                               \
  } while (0)

static thread_local void* t_seen = nullptr;

extern "C" {
int rafhip_device_count(void) { return 1; }
const char* rafhip_last_error(void) { return "stand-in"; }
int rafhip_sgd(const void*, const void*, const void*, void*, void*, int64_t, int32_t, double, double, void* stream) {
  t_seen = stream;
  return RAFHIP_OK;
}
int rafhip_embedding(const void*, int32_t, int64_t, int64_t, const void*, int32_t, int64_t, int64_t, float, void*, int32_t,
                     void* stream) {
  t_seen = stream;
  return RAFHIP_OK;
}
int64_t rafhip_embedding_dx_workspace_bytes(int64_t, int64_t, int64_t) { return -1; }
int rafhip_embedding_dx(const void*, int32_t, const void*, int32_t, int64_t, int64_t, int64_t, int64_t, int32_t, int64_t, float,
                        void*, int32_t, int32_t, void*, int64_t, void*) {
  return RAFHIP_ERR_NO_DEVICE;
}
int64_t rafhip_topk_distill_workspace_bytes(const rafhip_topk_distill_args*) { return -1; }
int rafhip_topk_distill(const rafhip_topk_distill_args*, float*, float*, void*, int64_t, void*) { return RAFHIP_ERR_NO_DEVICE; }
int rafhip_topk_distill_dx(const rafhip_topk_distill_args*, const float*, int64_t, const float*, void*, int64_t, void*) {
  return RAFHIP_ERR_NO_DEVICE;
}
int rafhip_topk_distill_step(const rafhip_topk_distill_args*, const float*, int64_t, float*, void*, int64_t, void*, int64_t,
                             void*) {
  return RAFHIP_ERR_NO_DEVICE;
}
}  // extern "C"

static float g_memory[64];
static char g_streams[8];
static int64_t g_shape[2] = {4, 8}, g_ids_shape[1] = {4};

static rafhip_tensor_desc D(int slot, int32_t code = 2, int32_t bits = 32, int32_t ndim = 2, int64_t* shape = g_shape) {
  return rafhip_tensor_desc{&g_memory[slot], 10, 0, code, bits, ndim, shape};
}

static value::TensorValue T(int slot) {
  TensorView t;
  t.data = &g_memory[slot];
  t.shape = {4, 8};
  t.device = Device(DevType::kROCM(), 0);
  return value::MakeTensor(t);
}

int main() {
  const Device rocm(DevType::kROCM(), 0);
  auto api = device_api::DeviceAPI::Get(DevType::kROCM());
  auto on_a_thread = [&](auto&& f) { std::thread(f).join(); };

  std::puts("set on one thread, executed on another");
  auto args = std::make_shared<schema::SgdArgs>();
  args->x = T(0);
  args->dx = T(1);
  args->v = T(2);
  CallValues call = MakeCall("raf.op.sgd", args);
  RunDeclare(call);
  OpEnvPtr env((*OpEnvMaker::Get("raf.op.hip.sgd"))(call));
  EXPECT(!env->HasError());
  OpEnv::SetStreamForAllBackends(rocm, &g_streams[1]);
  void* there = nullptr;
  on_a_thread([&] {
    env->Execute(call);
    there = t_seen;
  });
  EXPECT(there == &g_streams[1]);
  on_a_thread([&] { OpEnv::SetStreamForAllBackends(rocm, &g_streams[2]); });
  env->Execute(call);
  EXPECT(t_seen == &g_streams[2]);

  std::puts("a call of the C window: its own stream, which is the process's setting afterwards");
  rafhip_raf_env *sgd = nullptr, *lookup = nullptr;
  rafhip_tensor_desc x = D(0), dx = D(1), v = D(2), v1 = D(3), x1 = D(4), ids = D(5, 0, 64, 1, g_ids_shape), y = D(6);
  EXPECT(rafhip_raf_sgd_make(&x, &dx, &v, 0.1, 0.9, &sgd) == 0);
  EXPECT(rafhip_raf_embedding_make(&x, &ids, 1.0, 0, 2, 32, &lookup) == 0);
  const rafhip_tensor_desc lookup_in[] = {x, ids};
  EXPECT(rafhip_raf_sgd_execute(sgd, &x, &dx, &v, &v1, &x1, &g_streams[3]) == 0);
  EXPECT(t_seen == &g_streams[3] && api->GetStream() == &g_streams[3]);
  on_a_thread([&] { there = api->GetStream(); });
  EXPECT(there == &g_streams[3]);
  OpEnv::SetStreamForAllBackends(rocm, &g_streams[4]);  // and is no longer once another is set
  EXPECT(api->GetStream() == &g_streams[4]);
  g_ids_shape[0] = 3;  // a call that fails leaves nothing behind either
  const rafhip_tensor_desc wrong = D(5, 0, 64, 1, g_ids_shape), wrong_in[] = {x, wrong};
  EXPECT(rafhip_raf_execute(lookup, 2, wrong_in, 1, &y, nullptr, 0, &g_streams[3]) != 0);
  g_ids_shape[0] = 4;
  OpEnv::SetStreamForAllBackends(rocm, &g_streams[4]);
  EXPECT(api->GetStream() == &g_streams[4]);

  std::puts("threads at once, each with its own stream, and one that keeps setting the process's");
  std::atomic<int> wrong_stream{0}, failed{0};
  std::atomic<bool> stop{false};
  std::thread setter([&] {
    while (!stop) OpEnv::SetStreamForAllBackends(rocm, &g_streams[7]);
  });
  std::vector<std::thread> threads;
  for (int k = 0; k < 4; ++k)
    threads.emplace_back([&, k] {
      rafhip_tensor_desc xk = x, dxk = dx, vk = v, v1k = v1, x1k = x1, yk = y;
      for (int i = 0; i < 20000; ++i) {
        const int status = k % 2 ? rafhip_raf_sgd_execute(sgd, &xk, &dxk, &vk, &v1k, &x1k, &g_streams[k])
                                 : rafhip_raf_execute(lookup, 2, lookup_in, 1, &yk, nullptr, 0, &g_streams[k]);
        failed += status != 0;
        wrong_stream += t_seen != &g_streams[k];
      }
    });
  for (auto& t : threads) t.join();
  stop = true;
  setter.join();
  EXPECT(failed == 0 && wrong_stream == 0);
  rafhip_raf_env_destroy(sgd);
  rafhip_raf_env_destroy(lookup);
  std::puts("ALL OK");
  return 0;
}
