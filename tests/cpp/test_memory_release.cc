// Stream-ordered memory and its end: freed on its stream, at once where the runtime refuses that, and
// never freed twice.  The runtime is a stand-in in which a stream can be gone and a pointer can be
// foreign (memory of a captured graph, say).
#include <cstdio>
#include <set>
#include <string>
#include <vector>

#include "rafhip_device.h"
#include "rafhip_dialect.h"
#include "rafhip_vocab.h"

#define EXPECT(cond)                                                \
  do {                                                              \
    if (!(cond)) {                                                  \
      std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
      return 1;                                                     \
    }                                                               \
  } while (0)

static std::set<void*> g_gone, g_live;
static std::vector<std::string> g_log;
static char g_memory[16];
static int g_next = 0;

extern "C" {
int rafhip_dev_set(int32_t) { return RAFHIP_OK; }
int rafhip_dev_alloc_async(int32_t, int64_t, void*, void** out) {
  *out = &g_memory[g_next++];
  g_live.insert(*out);
  return RAFHIP_OK;
}
int rafhip_dev_free_async(void* ptr, void* stream) {
  if (g_gone.count(stream) || !g_live.count(ptr)) return RAFHIP_ERR_HIP;
  g_live.erase(ptr);
  g_log.push_back("on the stream");
  return RAFHIP_OK;
}
int rafhip_dev_free(void* ptr) {
  if (!g_live.count(ptr)) return RAFHIP_ERR_HIP;
  g_live.erase(ptr);
  g_log.push_back("at once");
  return RAFHIP_OK;
}
// The operators at the vocabulary are linked in but not called.
int rafhip_embedding(const void*, int32_t, int64_t, int64_t, const void*, int32_t, int64_t, int64_t, float, void*, int32_t,
                     void*) {
  return RAFHIP_ERR_NO_DEVICE;
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

int main() {
  char streams[2];
  rafhip_raf_memory* mem[3] = {};
  for (int i = 0; i < 3; ++i) EXPECT(rafhip_raf_memory_alloc(10, 0, 100, 0, 1, &streams[i % 2], &mem[i]) == 0);
  EXPECT(g_live.size() == 3);

  EXPECT(rafhip_raf_memory_free(mem[0]) == 0);
  EXPECT(g_log == std::vector<std::string>{"on the stream"} && g_live.size() == 2);

  std::puts("the stream is gone: freed all the same");
  g_gone.insert(&streams[1]);
  EXPECT(rafhip_raf_memory_free(mem[1]) == 0);
  EXPECT((g_log == std::vector<std::string>{"on the stream", "at once"}) && g_live.size() == 1);

  std::puts("memory that is not the caller's any more: reported, and nothing is thrown");
  g_live.clear();
  EXPECT(rafhip_raf_memory_free(mem[2]) == 0);
  EXPECT(g_log.size() == 2);
  std::puts("ALL OK");
  return 0;
}
