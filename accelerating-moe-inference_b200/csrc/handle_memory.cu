// Device memory of the 4-bit operators' handles (handle_alloc, handle_free in
// dtype.cuh).
//
// cudaMalloc costs 0.3 to 0.8 ms whatever its size, which is most of what a small
// handle costs to make, and a model has a handle for each of its matrices.  So
// handles of up to 64 MB share slabs, first fit; larger ones have allocations of
// their own.  A block goes back only after the device has finished what was
// enqueued before, as with cudaFree; of slabs without blocks the largest is kept.
// Making and closing a cache handle: 0.012 + 0.002 ms (0.34 + 0.27 with an
// allocation of its own), one for 2048 x 2048 weights 0.022 + 0.003 (0.36 + 0.28).
#include <algorithm>
#include <iterator>
#include <map>
#include <memory>
#include <mutex>
#include <vector>

#include "dtype.cuh"

namespace moe {
namespace {

constexpr size_t kAlign = 1024, kSlabStep = 32ull << 20, kShared = 64ull << 20;

struct Slab {
    int device = 0;
    uint8_t* base = nullptr;
    size_t bytes = 0;
    std::map<size_t, size_t> free;    // offset -> bytes, no two adjacent
    bool empty() const { return free.size() == 1 && free.begin()->second == bytes; }
};

struct Block {
    Slab* slab = nullptr;             // null: an allocation of its own
    size_t at = 0, bytes = 0;
};

struct Memory {
    std::mutex mutex;
    std::vector<std::unique_ptr<Slab>> slabs;
    std::map<void*, Block> used;
};

Memory& memory() {
    static Memory* m = new Memory;    // not destroyed: handles may be, at the process's end
    return *m;
}

// `bytes` of a slab that has room, or null.
void* take(Memory& m, Slab* s, size_t bytes) {
    for (auto it = s->free.begin(); it != s->free.end(); ++it) {
        if (it->second < bytes) continue;
        const size_t at = it->first, left = it->second - bytes;
        void* p = s->base + at;
        m.used.emplace(p, Block{s, at, bytes});
        if (left) {                   // the range's node moves to its rest
            auto node = s->free.extract(it);
            node.key() = at + bytes;
            node.mapped() = left;
            s->free.insert(std::move(node));
        } else {
            s->free.erase(it);
        }
        return p;
    }
    return nullptr;
}

}  // namespace

cudaError_t handle_alloc(int device, size_t bytes, void** out) {
    Memory& m = memory();
    std::lock_guard<std::mutex> lock(m.mutex);
    bytes = std::max(kAlign, (bytes + kAlign - 1) / kAlign * kAlign);
    if (bytes <= kShared) {
        for (auto& s : m.slabs)
            if (s->device == device && (*out = take(m, s.get(), bytes))) return cudaSuccess;
        auto s = std::make_unique<Slab>();
        s->device = device;
        s->bytes = std::max(kSlabStep, (4 * bytes + kSlabStep - 1) / kSlabStep * kSlabStep);
        s->free.emplace(0, s->bytes);
        m.slabs.reserve(m.slabs.size() + 1);
        if (cudaMalloc(&s->base, s->bytes) == cudaSuccess) {
            m.slabs.push_back(std::move(s));
            *out = take(m, m.slabs.back().get(), bytes);
            return cudaSuccess;
        }
        cudaGetLastError();           // no room for a slab: the block alone may still fit
    }
    auto it = m.used.emplace(nullptr, Block{nullptr, 0, bytes}).first;
    void* p = nullptr;
    const cudaError_t e = cudaMalloc(&p, bytes);
    auto node = m.used.extract(it);
    if (e != cudaSuccess) return e;
    node.key() = p;
    m.used.insert(std::move(node));
    *out = p;
    return cudaSuccess;
}

void handle_free(void* p) noexcept {
    if (!p) return;
    // What was enqueued with it has to be done.  Where that cannot be known (inside
    // a capture, after a fault) the block stays taken.
    if (cudaDeviceSynchronize() != cudaSuccess) {
        cudaGetLastError();
        return;
    }
    Memory& m = memory();
    std::lock_guard<std::mutex> lock(m.mutex);
    const auto it = m.used.find(p);
    if (it == m.used.end()) return;
    const Block b = it->second;
    if (!b.slab) {
        m.used.erase(it);
        cudaFree(p);
        return;
    }
    auto& free = b.slab->free;
    try {
        free.emplace(b.at, b.bytes);
    } catch (...) {
        return;                       // no memory for the note: the block stays taken
    }
    m.used.erase(it);
    auto here = free.find(b.at);
    if (const auto next = std::next(here); next != free.end() && here->first + here->second == next->first) {
        here->second += next->second;
        free.erase(next);
    }
    if (here != free.begin())
        if (const auto before = std::prev(here); before->first + before->second == here->first) {
            before->second += here->second;
            free.erase(here);
        }
    if (!b.slab->empty()) return;
    // The largest of the device's slabs without blocks stays.
    auto least = m.slabs.end();
    int empty = 0;
    for (auto s = m.slabs.begin(); s != m.slabs.end(); ++s) {
        if ((*s)->device != b.slab->device || !(*s)->empty()) continue;
        ++empty;
        if (least == m.slabs.end() || (*s)->bytes < (*least)->bytes) least = s;
    }
    if (empty < 2) return;
    cudaFree((*least)->base);
    m.slabs.erase(least);
}

}  // namespace moe
