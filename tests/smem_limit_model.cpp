// Two threads' first launches of one kernel, one with 100 KB and one with 60 KB of shared memory, with every order of what
// they do to the kernel's limit: the first thread's change is held back until the second one has come as far.
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <initializer_list>
#include <mutex>
#include <thread>

#include "smem_limit.h"

static int run(bool larger_first) {
  slora::SmemLimit limit;
  std::mutex m;
  std::condition_variable cv;
  size_t set_to = 0;
  int calls = 0;
  auto launch = [&](size_t smem) {
    return limit.allow(0, smem, [] { return size_t(200) << 10; }, [&](size_t bytes) {
      std::unique_lock<std::mutex> lock(m);
      set_to = bytes;
      ++calls;
      cv.notify_all();
      cv.wait_for(lock, std::chrono::seconds(1), [&] { return calls > 1; });
      return true;
    });
  };
  const size_t a = size_t(larger_first ? 100 : 60) << 10, b = size_t(larger_first ? 60 : 100) << 10;
  bool ok_a = false, ok_b = false;
  std::thread one([&] { ok_a = launch(a); });
  {
    std::unique_lock<std::mutex> lock(m);
    cv.wait_for(lock, std::chrono::seconds(1), [&] { return calls > 0; });
  }
  std::thread two([&] { ok_b = launch(b); });
  one.join();
  two.join();
  int bad = !ok_a || !ok_b;
  for (size_t kb : {20, 60, 100, 200}) {
    if (!launch(kb << 10) || (kb > 48 && set_to < kb << 10)) {
      printf("%s first: a launch with %zu KB finds a limit of %zu KB\n", larger_first ? "larger" : "smaller", kb, set_to >> 10);
      bad = 1;
    }
  }
  return bad;
}

int main() {
  int bad = run(true) + run(false);
  slora::SmemLimit limit;
  if (limit.allow(1, 100 << 10, [] { return size_t(200) << 10; }, [](size_t) { return false; })) bad = 1;  // a refusal is passed on
  int sets = 0;
  for (int i = 0; i < 3; ++i) limit.allow(1, 100 << 10, [] { return size_t(200) << 10; }, [&](size_t) { return ++sets > 0; });
  if (sets != 1) bad = 1;                                                                                   // and tried again, once
  for (int i = 0; i < 3; ++i) limit.allow(-1, 100 << 10, [] { return size_t(200) << 10; }, [&](size_t) { return ++sets > 0; });
  if (sets != 4) bad = 1;
  return bad;
}
