// Calls of one entry point from several native threads at once, for the tests of the GPU library (Python's own
// threads take turns).
#include <atomic>
#include <cstdint>
#include <thread>
#include <vector>

extern "C" {

// tk_kv4_gather_async
typedef int (*gather_fn)(void* dev, const void* cache, const int32_t* slots, void* k, void* v, uint32_t tokens,
                         uint32_t k_stride, uint32_t v_stride, int dtype, void* stream);

// `calls` calls from each of `threads` threads, thread i with keys[i], values[i], streams[i]; the number that failed.
int gather_from_threads(gather_fn gather, void* dev, const void* cache, const int32_t* slots, void** keys, void** values,
                        void** streams, int threads, int calls) {
  std::atomic<int> ready{0}, failed{0};
  std::vector<std::thread> all;
  for (int i = 0; i < threads; ++i)
    all.emplace_back([&, i] {
      ++ready;
      while (ready.load() < threads) std::this_thread::yield();
      for (int c = 0; c < calls; ++c)
        if (gather(dev, cache, slots, keys[i], values[i], 1, 0, 0, 0, streams[i]) != 0) ++failed;
    });
  for (auto& t : all) t.join();
  return failed.load();
}
}
