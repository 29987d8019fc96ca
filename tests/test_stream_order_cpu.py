"""The host lock that keeps the launches of one call together on its stream (csrc/stream_order.h), compiled
and run without CUDA: two threads' calls on one stream do not mix, other streams do not wait, and the per-thread
handle stands for another stream in every thread."""
import os
import subprocess

from tests.conftest import ROOT

PROGRAM = r"""
#include "stream_order.h"

#include <cstdio>
#include <thread>

using namespace b200q8;
using Table = PerStream<int>;

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

int main()
{
    const void *a = (const void*)0x10, *b = (const void*)0x20, *per_thread = (const void*)2;
    Table table;

    // A "call" queues three launches; the queue's order must hold them together.
    std::vector<int> queue;
    std::mutex queue_mu;
    std::atomic<int> ready{0};
    auto caller = [&](int id) {
        ready++;
        while (ready < 2) std::this_thread::yield();
        for (int i = 0; i < 3000; i++) {
            Table::Held h;
            table.hold(stream_key(0, a, per_thread), &h);
            table.hold(stream_key(0, a, per_thread), &h);  // held already: no second wait
            ++*h;
            for (int launch = 0; launch < 3; launch++) {
                std::lock_guard<std::mutex> lk(queue_mu);
                queue.push_back(id);
                if (i % 7 == launch) std::this_thread::yield();
            }
        }
    };
    std::thread t1(caller, 1), t2(caller, 2);
    t1.join(), t2.join();
    CHECK(queue.size() == 2 * 3 * 3000);
    for (size_t i = 0; i < queue.size(); i += 3) CHECK(queue[i] == queue[i + 1] && queue[i] == queue[i + 2]);
    Table::Held h;
    table.hold(stream_key(0, a, per_thread), &h);
    CHECK(*h == 6000);

    // Another stream, and the same handle on another device, are there while the first is held.
    bool other = false;
    std::thread([&] {
        Table::Held x, y;
        table.hold(stream_key(0, b, per_thread), &x);
        table.hold(stream_key(1, a, per_thread), &y);
        other = *x == 0 && *y == 0;
    }).join();
    CHECK(other);

    // Going on to another stream lets go of the first.
    table.hold(stream_key(0, b, per_thread), &h);
    bool free_again = false;
    std::thread([&] {
        Table::Held x;
        table.hold(stream_key(0, a, per_thread), &x);
        free_again = *x == 6000;
    }).join();
    CHECK(free_again);

    // Keys: one for a handle in all threads, but one a thread for the per-thread handle.
    const StreamKey mine = stream_key(0, per_thread, per_thread), plain = stream_key(0, a, per_thread);
    CHECK(mine == stream_key(0, per_thread, per_thread));
    StreamKey theirs, theirs_plain;
    std::thread([&] { theirs = stream_key(0, per_thread, per_thread), theirs_plain = stream_key(0, a, per_thread); }).join();
    CHECK(!(theirs == mine) && theirs_plain == plain);
    StreamKey later;  // a thread that comes after one that ended
    std::thread([&] { later = stream_key(0, per_thread, per_thread); }).join();
    CHECK(!(later == mine) && !(later == theirs));

    int entries = 0;
    h = Table::Held();
    table.for_each([&](const StreamKey&, int&) { entries++; });
    CHECK(entries == 3);
    std::puts("ok");
}
"""


def test_calls_on_one_stream_do_not_mix(tmp_path):
    src, exe = tmp_path / "order.cc", tmp_path / "order"
    src.write_text(PROGRAM)
    csrc = os.path.join(ROOT, "vvllm_b200", "csrc")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Werror", f"-I{csrc}", str(src), "-o", str(exe), "-pthread"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
