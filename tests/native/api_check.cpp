// Host check of the C ABI (aegean-tge_amd/csrc/tge_api.cpp) over a stand-in
// for the HIP runtime with two devices (fake_hip/hip/hip_runtime.h) and for the
// kernels' launchers, built with the address and undefined-behaviour
// sanitizers by tests/test_host_api.py. The launchers check that every buffer
// of the library that a launch would touch is on the current device.
//   devices  calls on an e4m3 pool with a plan made on another device are
//            refused, for a pool of the same shape, too; a batch planned anew on
//            another device has its buffers there
//   memory   host memory that runs out anywhere in tge_batch_plan comes back as
//            TGE_ERR_CAPACITY, no exception leaves the call, the batch has no
//            plan, and the same plan succeeds afterwards
// Prints "api_check ok" or the first failure (exit 1).
#include <cstdio>
#include <cstdlib>
#include <new>
#include <string>
#include <vector>

#include "../../aegean-tge_amd/csrc/e4m3_kernels.h"
#include "../../aegean-tge_amd/csrc/tge_kernels.h"
#include "tge_kv.h"

#define REQUIRE(c, ...)                                        \
  do {                                                         \
    if (!(c)) {                                                \
      std::printf("FAIL %s:%d: %s: ", __FILE__, __LINE__, #c); \
      std::printf(__VA_ARGS__);                                \
      std::printf("\n");                                       \
      std::exit(1);                                            \
    }                                                          \
  } while (0)

// ---- host memory that runs out at the n-th allocation ------------------------------
namespace {
long g_until_failure = -1;  // allocations that still succeed (-1: all)
void* allocate(std::size_t n) {
  if (g_until_failure == 0) throw std::bad_alloc();
  if (g_until_failure > 0) --g_until_failure;
  void* p = std::malloc(n ? n : 1);
  if (!p) throw std::bad_alloc();
  return p;
}
}  // namespace
void* operator new(std::size_t n) { return allocate(n); }
void* operator new[](std::size_t n) { return allocate(n); }
void* operator new(std::size_t n, const std::nothrow_t&) noexcept {
  return g_until_failure == 0 ? nullptr : std::malloc(n ? n : 1);
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete[](void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }
void operator delete[](void* p, std::size_t) noexcept { std::free(p); }

// ---- the launchers --------------------------------------------------------------
namespace {
int g_launches = 0;
void here(const void* p, const char* what) {
  const int now = fake_hip::state().device, at = fake_hip::owner(p);
  REQUIRE(at == now, "%s of a launch on device %d is on device %d", what, now, at);
}
}  // namespace

namespace tge {
hipError_t launch_e4m3_append(const E4m3Append& p, hipStream_t) {
  here(p.blocks, "pool");
  here(p.tiles, "tiles");
  here(p.rows, "rows");
  return ++g_launches, hipSuccess;
}
hipError_t launch_e4m3_gather(const E4m3Gather& p, hipStream_t) {
  here(p.blocks, "pool");
  here(p.table, "table");
  return ++g_launches, hipSuccess;
}
hipError_t launch_e4m3_attention(int, int, const E4m3Attn& p, hipStream_t) {
  here(p.blocks, "pool");
  here(p.items, "items");
  here(p.tables, "tables");
  here(p.part_o, "partial states");
  here(p.part_ml, "partial sums");
  return ++g_launches, hipSuccess;
}
int e4m3_groups_per_cu(int width) { return width > 128 ? 1 : width > 64 ? 2 : 3; }
hipError_t launch_upload(char* dst, const char* src, std::size_t n, hipStream_t) {
  here(dst, "plan image");
  return std::memcpy(dst, src, n), hipSuccess;
}
hipError_t launch_kv_append(int, const AppendParams&, hipStream_t) { return ++g_launches, hipSuccess; }
hipError_t launch_kv_append_rope(int, const AppendParams&, hipStream_t) { return ++g_launches, hipSuccess; }
hipError_t launch_attention_group(int, int, int, const GroupParams&, hipStream_t) { return hipSuccess; }
hipError_t launch_kv_gather(int, const GatherParams&, hipStream_t) { return hipSuccess; }
hipError_t launch_step(int, int, int, int, int, const StepParams& p, hipStream_t) {
  here(p.recs, "step records");
  here(p.part_o, "partial states");
  here(p.counters, "counters");
  return ++g_launches, hipSuccess;
}
hipError_t launch_decode(int, int, int, int, int, const AttnParams& p, hipStream_t) {
  here(p.work, "work");
  here(p.part_o, "partial states");
  return ++g_launches, hipSuccess;
}
hipError_t launch_mixed(int, int, int, int, int, int, const AttnParams& a, const AttnParams& b, hipStream_t) {
  here(a.work, "work");
  here(b.work, "work");
  here(a.counters, "counters");
  return ++g_launches, hipSuccess;
}
int prefill_halves(int, int) { return 1; }
hipError_t launch_prefill(int, int, int, int, int, const AttnParams& p, hipStream_t) {
  here(p.work, "work");
  return ++g_launches, hipSuccess;
}
int decode_blocks_per_cu(int, int, int, int, bool) { return 2; }
int decode_app_waves(int, int, int, int) { return 0; }
hipError_t launch_reduce(int, int, int, const ReduceParams& p, hipStream_t) {
  here(p.items, "reduction records");
  return hipSuccess;
}
hipError_t read_wait_expiries(unsigned int*) { return hipSuccess; }
hipError_t launch_read_ceiling(const void*, std::size_t, int, int, int, hipStream_t) { return hipSuccess; }
}  // namespace tge

namespace {

void on(int device) { (void)hipSetDevice(device); }

struct Sessions {
  std::vector<int> ctx, n_new, offsets{0}, ids;
  Sessions(std::vector<std::pair<int, int>> s) {
    int page = 0;
    for (auto [c, n] : s) {
      ctx.push_back(c);
      n_new.push_back(n);
      for (int i = 0; i < (c + n + 15) / 16; ++i) ids.push_back(page++);
      offsets.push_back(page);
    }
  }
  tge_batch_desc desc(int q_heads) const {
    tge_batch_desc d{};
    d.n_sessions = (int)ctx.size();
    d.ctx = ctx.data();
    d.n_new = n_new.data();
    d.table_offsets = offsets.data();
    d.page_ids = ids.data();
    d.q_heads = q_heads;
    return d;
  }
};

tge_kv_pool* pool_on(int device, int format) {
  on(device);
  tge_kv_pool_desc d{};
  d.layers = 1;
  d.pages = 700;
  d.kv_heads = 2;
  d.head_dim = 128;
  d.format = format;
  tge_kv_pool* p = nullptr;
  REQUIRE(tge_kv_pool_create(&d, &p) == TGE_OK, "%s", tge_last_error());
  return p;
}

void check_devices() {
  const Sessions s({{9000, 2}, {40, 1}});
  const tge_batch_desc d = s.desc(8);
  alignas(16) static float x[4096];
  std::vector<char> codes(1 << 16);
  tge_append_rows_args store{};
  store.k = store.v = x;
  tge_attention_rows_args attend{};
  attend.q = attend.out = x;
  tge_kv_pool* pool[2] = {pool_on(0, TGE_KV_E4M3), pool_on(1, TGE_KV_E4M3)};
  tge_kv_pool* f16[2] = {pool_on(0, TGE_KV_F16), pool_on(1, TGE_KV_F16)};
  tge_batch* b = nullptr;
  REQUIRE(tge_batch_create(&b) == TGE_OK, "create");
  auto calls = [&](tge_kv_pool* p, int want, const char* what) {
    auto one = [&](const char* who, int got) {
      REQUIRE(got == want, "%s, %s: status %d (%s)", what, who, got, tge_last_error());
    };
    one("append_rows", tge_kv_append_rows(b, p, 0, &store, nullptr));
    one("attention_rows", tge_attention_rows(b, p, 0, &attend, nullptr));
    one("append", tge_kv_append(b, p, 0, x, x, nullptr));
    one("decode", tge_decode_attention(b, p, 0, x, x, nullptr));
    one("step", tge_decode_step(b, p, 0, x, x, x, x, nullptr));
    one("prefill", tge_prefill_attention(b, p, 0, x, x, nullptr));
    one("attention", tge_batch_attention(b, p, 0, x, x, nullptr));
    one("gather", tge_kv_gather(b, p, 0, 1, 16, codes.data(), codes.data(), codes.data(), codes.data(), nullptr));
  };
  for (int format : {TGE_KV_E4M3, TGE_KV_F16, TGE_KV_E4M3})
    for (int dev : {0, 1, 1, 0, 1}) {
      on(dev);
      tge_kv_pool* const mine = (format == TGE_KV_F16 ? f16 : pool)[dev];
      const int status = tge_batch_plan(b, mine, &d, nullptr);
      REQUIRE(status == TGE_OK, "%s", tge_last_error());
      if (format == TGE_KV_F16) {
        REQUIRE(tge_decode_step(b, mine, 0, x, x, x, x, nullptr) == TGE_OK, "%s", tge_last_error());
        REQUIRE(tge_prefill_attention(b, mine, 0, x, x, nullptr) == TGE_OK, "%s", tge_last_error());
        continue;
      }
      calls(mine, TGE_OK, "on the plan's device");
      const int before = g_launches;
      on(1 - dev);
      calls(mine, TGE_ERR_INVALID, "the current device is another one");
      calls(pool[1 - dev], TGE_ERR_INVALID, "the plan is on another device");
      on(dev);
      calls(pool[1 - dev], TGE_ERR_INVALID, "the pool is on another device");
      REQUIRE(g_launches == before, "a refused call launched");
    }
  // a plan that is refused leaves nothing to call
  on(0);
  REQUIRE(tge_batch_plan(b, pool[1], &d, nullptr) == TGE_ERR_INVALID, "plan for another device's pool");
  calls(pool[0], TGE_ERR_INVALID, "after a refused plan");
  fake_hip::state().capturing = true;
  REQUIRE(tge_batch_plan(b, pool[0], &d, nullptr) == TGE_ERR_INVALID, "plan while capturing");
  fake_hip::state().capturing = false;
  tge_batch_destroy(b);
  for (int i : {0, 1}) {
    tge_kv_pool_destroy(pool[i]);
    tge_kv_pool_destroy(f16[i]);
  }
  REQUIRE(fake_hip::state().live.empty(), "%zu allocations left", fake_hip::state().live.size());
}

void check_memory() {
  // (a decoding step cut into pieces, a prompt, both)
  for (const Sessions& s : {Sessions({{9000, 2}, {40, 1}}), Sessions({{100, 300}}), Sessions({{3000, 1}, {0, 200}})})
    for (int format : {TGE_KV_E4M3, TGE_KV_F16, TGE_KV_I8}) {
      const tge_batch_desc d = s.desc(8);
      alignas(16) static float x[4096];
      tge_kv_pool* pool = pool_on(0, format);
      int failures = 0;
      for (long n = 0;; ++n) {
        tge_batch* b = nullptr;
        REQUIRE(tge_batch_create(&b) == TGE_OK, "create");
        g_until_failure = n;
        int status = TGE_OK;
        bool left = false;
        try {
          status = tge_batch_plan(b, pool, &d, nullptr);
        } catch (...) {
          left = true;
        }
        const bool all = g_until_failure > 0;  // (the plan needed fewer)
        g_until_failure = -1;
        REQUIRE(!left, "format %d: an exception left the plan at allocation %ld", format, n);
        if (status != TGE_OK) {
          REQUIRE(status == TGE_ERR_CAPACITY, "format %d, allocation %ld: status %d", format, n, status);
          REQUIRE(std::string(tge_last_error()).find("memory") != std::string::npos, "%s", tge_last_error());
          REQUIRE(tge_kv_append(b, pool, 0, x, x, nullptr) == TGE_ERR_INVALID, "a call after a failed plan");
          REQUIRE(tge_batch_plan(b, pool, &d, nullptr) == TGE_OK, "%s", tge_last_error());
          ++failures;
        }
        REQUIRE(tge_kv_append(b, pool, 0, x, x, nullptr) == TGE_OK, "%s", tge_last_error());
        tge_batch_destroy(b);
        if (all) break;
      }
      REQUIRE(failures > 5, "%d failures", failures);
      tge_kv_pool_destroy(pool);
    }
}

}  // namespace

int main(int argc, char** argv) {
  const std::string which = argc > 1 ? argv[1] : "";
  if (which == "devices")
    check_devices();
  else if (which == "memory")
    check_memory();
  else
    REQUIRE(false, "unknown check");
  std::printf("api_check ok\n");
  return 0;
}
