// The turns that entry points take on a stream: a whole turn keeps other threads' calls on
// the same stream out, on streams of any origin, and nothing else.  Handles here are only
// numbers: no device is needed.  Prints "ok".
#include "../fast-llm_amd/csrc/flh_internal.h"
#include <atomic>
#include <chrono>
#include <cstdio>
#include <future>
#include <thread>
#include <vector>
using flh::StreamTurn;
using namespace std::chrono_literals;

static int fails = 0;
static void want(bool ok, const char * what, void * s) {
    if (ok) return;
    ++fails;
    std::printf("FAILED: %s (stream %p)\n", what, s);
}
// whether another thread gets a turn on `s` within `t`; it is given back at once.  A thread
// that is kept out goes on waiting: settle() joins them all, once nothing holds them.
static std::vector<std::thread> waiting;
static bool enters(void * s, bool whole, std::chrono::milliseconds t) {
    auto p = std::make_shared<std::promise<void>>();
    auto got = p->get_future();
    waiting.emplace_back([=] { { StreamTurn turn(s, whole); } p->set_value(); });
    return got.wait_for(t) == std::future_status::ready;
}
static void settle() {
    for (auto & t : waiting) t.join();
    waiting.clear();
}

int main() {
    void * const streams[] = {nullptr, (void *)2, (void *)0x7000, (void *)0x7fff12345678};
    for (void * s : streams) {
        {
            const StreamTurn replay(s, true);
            want(replay.device() == -1, "a stream made elsewhere has no device here", s);
            want(!enters(s, false, 150ms), "a call waits for a replay", s);
            want(!enters(s, true, 150ms), "a replay waits for a replay", s);
            for (void * o : streams)
                if (o != s) want(enters(o, true, 5000ms), "streams do not wait for one another", o);
        }
        settle();
        want(enters(s, true, 5000ms), "the turn ends", s);
        {
            const StreamTurn call(s);
            want(enters(s, false, 5000ms), "calls do not exclude each other", s);
            want(!enters(s, true, 150ms), "a replay waits for a call", s);
        }
        settle();
    }
    // many streams that come and go, while one is held
    {
        const StreamTurn held((void *)0x9000, true);
        for (uintptr_t i = 1; i <= 20000; ++i) StreamTurn turn((void *)(0x100000 + 64 * i), i % 3 == 0);
        want(!enters((void *)0x9000, false, 150ms), "a held turn is kept", (void *)0x9000);
    }
    settle();
    if (!fails) std::puts("ok");
    return fails != 0;
}
