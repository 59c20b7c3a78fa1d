// test_stream_order.cpp -- the order of a context's calls (vq_b200/csrc/stream_order.hpp) over streams that are sets of jobs.  Built and run by tests/test_stream_order.py.
#include <cstdio>
#include <random>
#include <set>
#include <vector>

#include "../../vq_b200/csrc/stream_order.hpp"

static int failed = 0;
static const char *scene = "";

constexpr int OWN = 0, DEFAULT = 1, STREAMS = 5; // 0: the context's own stream, 1: the default stream, others the caller's

struct Fake {
    using Stream = int;
    std::vector<std::set<int>> seen = std::vector<std::set<int>>(STREAMS); // jobs that whatever comes next on a stream runs behind
    std::set<int> event;
    bool in_capture[STREAMS] = {};
    bool blocking = false; // the captured stream is one that the default stream waits for: the default stream cannot be asked
    bool lasting(int s) const { return s <= DEFAULT; }
    bool captured(int s) const
    {
        if (s == DEFAULT && blocking)
            for (int i = 2; i < STREAMS; ++i)
                if (in_capture[i]) return true;
        return in_capture[s];
    }
    void check(int s, const char *what) const
    {
        if (captured(s)) std::printf("FAIL %s: %s a captured stream\n", scene, what), ++failed;
    }
    void record(int s) { check(s, "recorded on"), event = seen[s]; }
    void wait(int s) { check(s, "waited on"), seen[s].insert(event.begin(), event.end()); }
};

// A context as CudaDevice uses the order.
struct Model {
    vqb::StreamOrder<Fake> order;
    int stream = OWN, jobs = 0;
    std::set<int> open; // eager jobs that the host has not waited for
    // An eager call, or, where its stream is being captured, one that becomes part of the graph.
    void call(int s, bool host_waits = false)
    {
        Fake &f = order.api;
        if (s == DEFAULT && f.captured(s)) return; // (CUDA would refuse it)
        const int old = stream;
        stream = s;
        order.change(old, s);
        order.call_ends(s); // (setting a stream is a call, too)
        order.settle(s);
        if (!f.captured(s)) {
            for (int j : open)
                if (!f.seen[s].count(j) && !(f.blocking && f.captured(DEFAULT))) std::printf("FAIL %s: a call on stream %d is not behind job %d\n", scene, s, j), ++failed;
            f.seen[s].insert(++jobs);
            open.insert(jobs);
        }
        order.launched();
        if (host_waits && !f.captured(s)) {
            order.waited();
            const std::set<int> done = f.seen[s];
            for (int j : done) open.erase(j);
        }
        order.call_ends(s);
    }
    void capture(int s) { order.api.in_capture[s] = true; }
    void end_capture(int s) { order.api.in_capture[s] = false; }
};

int main()
{
    {
        scene = "the capture's own stream";
        Model m;
        m.call(2);
        m.capture(3), m.call(3), m.end_capture(3);
        m.call(3);
    }
    {
        scene = "a third stream";
        Model m;
        m.call(2);
        m.capture(3), m.call(3), m.end_capture(3);
        m.call(4);
    }
    {
        scene = "own stream, capture, its stream, another one";
        Model m;
        m.call(OWN);
        m.capture(3), m.call(3), m.call(3), m.end_capture(3);
        m.call(3), m.call(4), m.call(OWN), m.call(2);
    }
    {
        scene = "two captures before anything eager";
        Model m;
        m.call(2);
        m.capture(3), m.call(3), m.end_capture(3);
        m.capture(4), m.call(4), m.end_capture(4);
        m.call(4);
    }
    {
        scene = "a host wait on a stream that owes";
        Model m;
        m.call(2);
        m.capture(3), m.call(3, true), m.end_capture(3);
        m.call(3, true), m.call(4);
    }
    {
        scene = "the default stream before a capture that it cannot be asked in";
        Model m;
        m.order.api.blocking = true;
        m.call(DEFAULT);
        m.capture(3), m.call(3), m.end_capture(3);
        m.call(3), m.call(2);
    }
    scene = "any order";
    for (int seed = 0; seed < 20000 && !failed; ++seed) {
        std::mt19937 rng(seed);
        Model m;
        m.order.api.blocking = seed & 1;
        int captured = -1;
        for (int step = 0; step < 40; ++step) {
            const unsigned what = rng() % 10;
            if (captured < 0 && what == 0) m.capture(captured = 2 + rng() % (STREAMS - 2));
            else if (captured >= 0 && what <= 2) m.end_capture(captured), captured = -1;
            else m.call(rng() % STREAMS, what == 9);
        }
    }
    std::printf(failed ? "%d checks failed\n" : "all checks of the order of calls passed\n", failed);
    return failed != 0;
}
