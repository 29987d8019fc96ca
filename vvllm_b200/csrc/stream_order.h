// stream_order.h -- what calls on one CUDA stream share, one call at a time.  Host code without CUDA headers.
//
// A call may be several launches that meet in the stream's scratch.  The GPU runs them in the order in which they
// were queued, so that order must not mix two calls' launches: whoever uses the scratch holds its entry from
// the lookup to the last launch.  Calls of other streams do not wait.
#pragma once

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <functional>
#include <memory>
#include <mutex>
#include <unordered_map>
#include <utility>
#include <vector>

namespace b200q8 {

// A stream of a device.  The per-thread handle is one value for a stream of every host thread: `thread` tells them
// apart (numbers are not used again).  For all others it is 0.
struct StreamKey {
    int dev = 0;
    const void* stream = nullptr;
    unsigned long long thread = 0;
    bool operator==(const StreamKey& o) const { return dev == o.dev && stream == o.stream && thread == o.thread; }
};

inline StreamKey stream_key(int dev, const void* stream, const void* per_thread_handle)
{
    static std::atomic<unsigned long long> next{1};
    thread_local const unsigned long long self = next.fetch_add(1, std::memory_order_relaxed);
    return {dev, stream, stream == per_thread_handle ? self : 0};
}

struct StreamKeyHash {
    size_t operator()(const StreamKey& k) const
    {
        return std::hash<uintptr_t>()((uintptr_t)k.stream) * 31u + (size_t)k.dev * 7u + (size_t)k.thread;
    }
};

// One T per stream.  Entries stay where they are, for good.
template <class T>
class PerStream {
    struct Entry {
        std::mutex mu;
        T value;
    };
    std::mutex mu_;  // of the table; never held while an entry is waited for
    std::unordered_map<StreamKey, std::unique_ptr<Entry>, StreamKeyHash> table_;

    Entry& find(const StreamKey& k)
    {
        std::lock_guard<std::mutex> lk(mu_);
        std::unique_ptr<Entry>& e = table_[k];
        if (!e) e = std::make_unique<Entry>();
        return *e;
    }

public:
    // A stream's entry, this holder's alone while it lives.
    class Held {
        std::unique_lock<std::mutex> lk_;
        Entry* e_ = nullptr;
        StreamKey key_;
        friend class PerStream;

    public:
        explicit operator bool() const { return e_ != nullptr; }
        const StreamKey& key() const { return key_; }
        T& operator*() const { return e_->value; }
    };

    // Takes the entry of k; nothing to do where `h` holds it already.
    void hold(const StreamKey& k, Held* h)
    {
        if (h->e_ && h->key_ == k) return;
        *h = Held();
        Entry& e = find(k);
        h->lk_ = std::unique_lock<std::mutex>(e.mu);
        h->e_ = &e;
        h->key_ = k;
    }

    // f(key, value) for every entry, each held for its turn.
    template <class F>
    void for_each(F f)
    {
        std::unique_lock<std::mutex> lk(mu_);
        std::vector<std::pair<StreamKey, Entry*>> all;
        for (auto& kv : table_) all.emplace_back(kv.first, kv.second.get());
        lk.unlock();
        for (auto& [k, e] : all) {
            std::lock_guard<std::mutex> in(e->mu);
            f(k, e->value);
        }
    }
};

}  // namespace b200q8
