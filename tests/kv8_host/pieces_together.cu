// Runs the loop in which the 256-row kernel's converting warps take their pieces (pieces_together) with
// four threads for the four warps and a barrier that needs all of them. In each case one thread gives
// up, at the wait for a piece or inside it. Exit code 0: all four always left, and alike. A thread left at
// the barrier is seen by a time limit.
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <mutex>
#include <thread>

#include "kv8_attn.cuh"

struct Barrier {
  std::mutex m;
  std::condition_variable cv;
  int here = 0, round = 0;
  bool all = true, last = true, stuck = false;
  bool meet(bool ok) {  // whether all four are ok
    std::unique_lock<std::mutex> lock(m);
    all = all && ok;
    const int mine = round;
    if (++here == 4) {
      last = all;
      all = true;
      here = 0;
      ++round;
      cv.notify_all();
      return last;
    }
    if (!cv.wait_for(lock, std::chrono::seconds(2), [&] { return round != mine; })) {
      stuck = true;
      return false;
    }
    return last;
  }
};

// Thread `who` gives up at piece `piece`: at the wait for it (tile < 0) or in its tile `tile`.
static bool run(int who, int piece, int tile) {
  constexpr int PIECES = 3, TILES = 2;
  Barrier bar;
  bool ended[4];
  std::thread threads[4];
  for (int w = 0; w < 4; ++w) {
    threads[w] = std::thread([&, w] {
      int n = 0;
      auto next = [&]() -> int { return w == who && n == piece && tile < 0 ? -1 : n++ < PIECES ? 1 : 0; };
      auto agree = [&](bool ok) { return bar.meet(ok); };
      auto work = [&]() -> bool {
        for (int t = 0; t < TILES; ++t) {
          bar.meet(true);
          if (!bar.meet(!(w == who && n - 1 == piece && t == tile))) return false;
        }
        return true;
      };
      ended[w] = fa2kv::pieces_together(next, agree, work);
    });
  }
  for (auto& t : threads) t.join();
  bool good = !bar.stuck;
  for (int w = 0; w < 4; ++w) good = good && ended[w] == (who < 0);
  if (!good) std::printf("thread %d gives up at piece %d, tile %d: stuck %d\n", who, piece, tile, bar.stuck);
  return good;
}

int main() {
  bool good = run(-1, 0, 0);  // nobody gives up
  for (int who = 0; who < 4; ++who) {
    for (int piece = 0; piece <= 3; ++piece) {
      good = run(who, piece, -1) && good;
      if (piece < 3) good = run(who, piece, 0) && run(who, piece, 1) && good;
    }
  }
  return good ? 0 : 1;
}
