// Streams with weights that were just written (no CUDA in this file: tests/test_fresh.py walks through it with the host compiler).
#pragma once

#include <atomic>
#include <mutex>

namespace mtc {

// What runs and what a graph under capture records are apart, each with a list of its own: a captured product does not run, so the wait of
// one that does is not its to use up, and captures that end without a product fill up their own list only.  Locked: two threads may
// quantize and multiply on streams of their own.
class FreshWeights {
public:
    static constexpr int kMost = 64;

    // a quantizer of weights went to this stream
    void written(const void *stream, bool captured) {
        const std::lock_guard<std::mutex> hold(lock);
        if (!captured) drop(lists[1], stream);
        List &l = lists[captured];
        for (int i = 0; i < l.n; ++i)
            if (l.streams[i] == stream) return;
        if (l.n < kMost) l.streams[l.n++] = stream;
        else l.anywhere = true;
        something.store(true, std::memory_order_release);
    }
    // is there anything that a product would have to look up?
    bool known() const { return something.load(std::memory_order_acquire); }
    // may a product that goes to this stream start on its weights early?  The first one behind a quantizer may not, and is the one that waits.
    bool early(const void *stream, bool captured) {
        const std::lock_guard<std::mutex> hold(lock);
        if (!captured) drop(lists[1], stream);
        List &l = lists[captured];
        const bool fresh = drop(l, stream);
        const bool may = !fresh && !l.anywhere;
        something.store(lists[0].n || lists[1].n || lists[0].anywhere || lists[1].anywhere, std::memory_order_release);
        return may;
    }

private:
    struct List {
        int n = 0;
        bool anywhere = false;               // more streams than the list holds: no product of this kind starts early any more
        const void *streams[kMost] = {};
    };
    // (a stream that work goes to outside a capture is in no capture: what one left there is over, and whatever replays it is ordered behind it)
    static bool drop(List &l, const void *stream) {
        for (int i = 0; i < l.n; ++i)
            if (l.streams[i] == stream) {
                l.streams[i] = l.streams[--l.n];
                return true;
            }
        return false;
    }

    std::mutex lock;
    std::atomic<bool> something{false};
    List lists[2];                           // [captured]
};

}  // namespace mtc
