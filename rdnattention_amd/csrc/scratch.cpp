// Stream-ordered scratch memory for the attention calls (the RoPE-rotated K
// copy, split-K partials, quantiser partials, INT8 decode scores).
//
// The reference allocates nothing (src/c_api.hpp:3-6); its kernels need no
// scratch.  Here a call that needs scratch takes the buffer cached for its
// (device, stream, use) and touches no allocator once that buffer is large
// enough.  Measured on MI355X under ROCm 7: hipFree waits until the whole
// device is idle (~32 ms behind a busy stream, even for a buffer no kernel
// uses), while hipMalloc and the default pool's hipMallocAsync / hipFreeAsync
// return without waiting for the GPU.  So no call ever runs hipFree:
//   * a buffer that must grow is released with hipFreeAsync on the call's
//     stream (after the buffer's last use) and replaced with hipMallocAsync;
//   * the cached bytes of a device, over all streams and uses, are capped
//     (kDeviceCap); growth past the cap first evicts the least recently used
//     idle entries, released the same way in the calling stream's order
//     after their own last use (hipStreamWaitEvent on the event recorded
//     after it), and a call that still does not fit takes a per-call
//     default-pool block instead;
//   * buffers above kEntryMax are never cached, only taken per call;
//   * a captured call takes a block that its graph owns (GraphBlock) until the graph
//     and its executables are destroyed.  A memory node (hipMallocAsync under
//     capture) will not do: the runtime gives the nodes of one graph the
//     addresses of another's, so that two graphs replayed side by side on two streams
//     use one buffer, and the records read from it lead anywhere.  The address is part
//     of the graph: copies of it must not run at the same time, nor its last replay
//     behind its destruction.  These blocks are outside of the caps above.
// rdna_scratch_trim() (the one synchronising path) frees every idle entry and
// returns the default pool's free blocks to the device.
#include "fa_internal.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

namespace rdna_amd {
namespace {

constexpr size_t kEntryMax = size_t(256) << 20;  // largest cached buffer
constexpr size_t kDeviceCap = size_t(1) << 30;   // cached bytes per device, all streams and uses
constexpr size_t kGranule = size_t(2) << 20;     // cached buffers grow in 2 MiB steps

struct Entry {
    void* ptr = nullptr;
    size_t bytes = 0;
    hipEvent_t last_use = nullptr; // recorded on the entry's stream after each use
    bool busy = false;             // a call holds the buffer
    uint64_t tick = 0;             // last use, for LRU eviction
};

struct DeviceCache {
    std::map<std::pair<hipStream_t, int>, Entry> entries;
    size_t bytes = 0;      // sum of the entries' buffers
    uint64_t tick = 0;
    int64_t allocations = 0; // allocator calls made for this device (cache growth and per-call blocks)
};

std::mutex g_mu;
std::map<int, DeviceCache> g_devices; // guarded by g_mu

std::string hip_err(const char* what, hipError_t e) {
    return std::string(what) + ": " + hipGetErrorString(e);
}

// A failed hipMallocAsync: `err` and what alloc returns.  The error does not
// stay behind for the check after the next launch, which a caller that can do
// with less makes.
int alloc_failed(hipError_t e, std::string& err) {
    (void)hipGetLastError();
    err = hip_err("scratch allocation failed", e);
    return e == hipErrorOutOfMemory ? kScratchFull : -1;
}

// A captured call's scratch.  The calls that one capture makes on one stream run in turn
// and share a block per use, as eager calls share the stream's; the graph holds it by a
// user object, whose destructor hands it back for later captures.
struct GraphBlock {
    using Key = std::tuple<unsigned long long, hipStream_t, int>; // capture, stream, use
    Key key;
    void* ptr = nullptr;
    size_t bytes = 0;
    int device = 0;
    bool busy = false; // a call of the capture holds it
};
struct GraphBlocks {
    std::mutex mu;
    std::map<GraphBlock::Key, GraphBlock*> held; // of each key the last
    std::vector<GraphBlock*> free;
    std::map<int, std::pair<uint64_t, int64_t>> made; // by device: bytes and blocks, held and free
};
// Never destroyed: a graph may outlive the library's static objects.
GraphBlocks& graph_blocks() {
    static auto* const blocks = new GraphBlocks;
    return *blocks;
}

// Returns the blocks that no graph owns to the devices (device < 0: all of them).
void free_graph_blocks(int device) {
    GraphBlocks& g = graph_blocks();
    std::vector<GraphBlock*> blocks;
    {
        std::lock_guard<std::mutex> lock(g.mu);
        const auto kept = std::partition(g.free.begin(), g.free.end(), [&](const GraphBlock* b) {
            return device >= 0 && b->device != device;
        });
        blocks.assign(kept, g.free.end());
        g.free.erase(kept, g.free.end());
        for (const GraphBlock* b : blocks) {
            auto& made = g.made[b->device];
            made.first -= b->bytes;
            made.second--;
        }
    }
    for (GraphBlock* b : blocks) {
        (void)hipFree(b->ptr);
        delete b;
    }
}

// User object's destructor: no HIP calls here.
void graph_block_released(void* p) {
    GraphBlocks& g = graph_blocks();
    auto* const b = static_cast<GraphBlock*>(p);
    std::lock_guard<std::mutex> lock(g.mu);
    const auto it = g.held.find(b->key);
    if (it != g.held.end() && it->second == b) {
        g.held.erase(it);
    }
    b->busy = false;
    g.free.push_back(b);
}

// A block of at least `bytes` for a call that stream s captures.  0, or what
// StreamScratch::alloc returns.
int graph_block(size_t bytes, hipStream_t s, int use, int device, GraphBlock*& out, bool& allocated,
                std::string& err) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    hipGraph_t graph = nullptr;
    const hipGraphNode_t* deps = nullptr;
    size_t n_deps = 0;
    hipError_t e = hipStreamGetCaptureInfo_v2(s, &status, &id, &graph, &deps, &n_deps);
    if (e != hipSuccess || graph == nullptr) {
        err = hip_err("scratch allocation under capture failed",
                      e != hipSuccess ? e : hipErrorStreamCaptureInvalidated);
        return -1;
    }
    GraphBlocks& g = graph_blocks();
    GraphBlock* b = nullptr;
    const size_t want = (bytes + kGranule - 1) / kGranule * kGranule;
    {
        std::lock_guard<std::mutex> lock(g.mu);
        const auto it = g.held.find({id, s, use});
        if (it != g.held.end() && !it->second->busy && it->second->bytes >= bytes && it->second->device == device) {
            out = it->second;
            out->busy = true;
            return 0;
        }
        // the smallest that holds it, of up to twice the size: a graph keeps it for its life
        auto best = g.free.end();
        for (auto f = g.free.begin(); f != g.free.end(); ++f) {
            if ((*f)->device == device && (*f)->bytes >= bytes && (*f)->bytes <= 2 * want &&
                (best == g.free.end() || (*f)->bytes < (*best)->bytes)) {
                best = f;
            }
        }
        if (best != g.free.end()) {
            b = *best;
            g.free.erase(best);
        }
    }
    if (b == nullptr) {
        void* ptr = nullptr;
        hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed; // hipMalloc is no part of the capture
        e = hipThreadExchangeStreamCaptureMode(&mode);
        if (e == hipSuccess) {
            e = hipMalloc(&ptr, want);
            if (e == hipErrorOutOfMemory) {
                (void)hipGetLastError();
                free_graph_blocks(device);
                e = hipMalloc(&ptr, want);
            }
            (void)hipThreadExchangeStreamCaptureMode(&mode);
        }
        if (e != hipSuccess) {
            return alloc_failed(e, err);
        }
        allocated = true;
        b = new GraphBlock;
        b->ptr = ptr;
        b->bytes = want;
        b->device = device;
        std::lock_guard<std::mutex> lock(g.mu);
        auto& made = g.made[device];
        made.first += want;
        made.second++;
    }
    b->key = {id, s, use};
    b->busy = true;
    hipUserObject_t owner = nullptr;
    e = hipUserObjectCreate(&owner, b, graph_block_released, 1, hipUserObjectNoDestructorSync);
    if (e != hipSuccess) {
        graph_block_released(b);
    } else {
        e = hipGraphRetainUserObject(graph, owner, 1, hipGraphUserObjectMove);
        if (e != hipSuccess) {
            (void)hipUserObjectRelease(owner, 1); // hands the block back
        }
    }
    if (e != hipSuccess) {
        err = hip_err("scratch allocation under capture failed", e);
        return -1;
    }
    std::lock_guard<std::mutex> lock(g.mu);
    g.held[b->key] = b;
    out = b;
    return 0;
}

// Releases e's buffer in the order of stream s: after the work recorded in
// its last_use event (a GPU-side wait), then hipFreeAsync on s.  Nothing here
// waits on the host.
hipError_t release_in_order(Entry& e, hipStream_t s) {
    hipError_t r = hipSuccess;
    if (e.ptr != nullptr) {
        if (e.last_use != nullptr) {
            r = hipStreamWaitEvent(s, e.last_use, 0);
        }
        if (r == hipSuccess) {
            r = hipFreeAsync(e.ptr, s);
        }
    }
    e.ptr = nullptr;
    e.bytes = 0;
    return r;
}

} // namespace

int StreamScratch::alloc(size_t bytes, hipStream_t s, std::string& err) {
    stream = s;
    if (bytes == 0) {
        return 0;
    }
    if (region != nullptr) {
        const size_t take = region_bytes(bytes);
        if (region->used + take > region->bytes) {
            err = "scratch region exhausted (" + std::to_string(region->used + take) + " of " +
                  std::to_string(region->bytes) + " bytes)";
            return -1;
        }
        ptr = region->base + region->used;
        region->used += take;
        return 0;
    }
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) {
        err = hip_err("scratch allocation failed", e);
        return -1;
    }
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    e = hipStreamIsCapturing(s, &capture);
    if (e != hipSuccess) {
        err = hip_err("scratch allocation failed", e);
        return -1;
    }
    if (capture != hipStreamCaptureStatusNone) {
        GraphBlock* b = nullptr;
        bool allocated = false;
        const int rc = graph_block(bytes, s, static_cast<int>(use), device, b, allocated, err);
        if (allocated) {
            std::lock_guard<std::mutex> lock(g_mu);
            g_devices[device].allocations++;
        }
        if (rc == 0) {
            graph = b;
            ptr = b->ptr;
        }
        return rc;
    }
    bool per_call = bytes > kEntryMax;
    if (!per_call) {
        std::lock_guard<std::mutex> lock(g_mu);
        DeviceCache& dc = g_devices[device];
        const auto key = std::make_pair(s, static_cast<int>(use));
        Entry& ent = dc.entries[key];
        if (ent.busy) {
            // another host thread's call on this stream holds the buffer
            per_call = true;
        } else {
            if (ent.bytes < bytes) {
                const size_t want = std::min(kEntryMax, (bytes + kGranule - 1) / kGranule * kGranule);
                size_t total = dc.bytes - ent.bytes + want;
                // over the cap: evict idle entries, least recently used first
                while (total > kDeviceCap) {
                    auto victim = dc.entries.end();
                    for (auto it = dc.entries.begin(); it != dc.entries.end(); ++it) {
                        if (it->first != key && !it->second.busy && it->second.ptr != nullptr &&
                            (victim == dc.entries.end() || it->second.tick < victim->second.tick)) {
                            victim = it;
                        }
                    }
                    if (victim == dc.entries.end()) {
                        break;
                    }
                    const size_t freed = victim->second.bytes;
                    e = release_in_order(victim->second, s);
                    if (victim->second.last_use != nullptr) {
                        (void)hipEventDestroy(victim->second.last_use);
                    }
                    dc.entries.erase(victim);
                    dc.bytes -= freed;
                    total -= freed;
                    if (e != hipSuccess) {
                        err = hip_err("scratch eviction failed", e);
                        return -1;
                    }
                }
                if (total > kDeviceCap) {
                    per_call = true; // every other entry is in use: do not cache this one
                } else {
                    const size_t old = ent.bytes;
                    e = release_in_order(ent, s);
                    dc.bytes -= old;
                    if (e == hipSuccess) {
                        e = hipMallocAsync(&ent.ptr, want, s);
                        dc.allocations++;
                    }
                    if (e != hipSuccess) {
                        ent.ptr = nullptr;
                        return alloc_failed(e, err);
                    }
                    ent.bytes = want;
                    dc.bytes += want;
                }
            }
            if (!per_call) {
                if (ent.last_use == nullptr) {
                    // device-scope only: the event orders GPU work (stream waits
                    // and the trim's synchronisation before a stream-ordered
                    // free); a system-scope release at each record would write
                    // back the L2 after every attention kernel
                    e = hipEventCreateWithFlags(&ent.last_use, hipEventDisableTiming | hipEventDisableSystemFence);
                } else {
                    // after the buffer's previous use; a no-op when that use was
                    // on this same stream, and it orders a handle that now names
                    // a new stream
                    e = hipStreamWaitEvent(s, ent.last_use, 0);
                }
                if (e != hipSuccess) {
                    err = hip_err("scratch allocation failed", e);
                    return -1;
                }
                ent.busy = true;
                ent.tick = ++dc.tick;
                ptr = ent.ptr;
                cached = true;
                return 0;
            }
        }
    }
    e = hipMallocAsync(&ptr, bytes, s);
    {
        std::lock_guard<std::mutex> lock(g_mu);
        g_devices[device].allocations++;
    }
    if (e != hipSuccess) {
        ptr = nullptr;
        return alloc_failed(e, err);
    }
    pooled = true;
    return 0;
}

StreamScratch::~StreamScratch() {
    if (cached) {
        // every kernel that uses the buffer has been enqueued on `stream`
        std::lock_guard<std::mutex> lock(g_mu);
        Entry& ent = g_devices[device].entries[std::make_pair(stream, static_cast<int>(use))];
        (void)hipEventRecord(ent.last_use, stream);
        ent.busy = false;
    } else if (pooled && ptr != nullptr) {
        (void)hipFreeAsync(ptr, stream);
    } else if (graph != nullptr) {
        std::lock_guard<std::mutex> lock(graph_blocks().mu);
        static_cast<GraphBlock*>(graph)->busy = false;
    }
}

int scratch_trim(std::string& err) {
    free_graph_blocks(-1);
    std::lock_guard<std::mutex> lock(g_mu);
    if (g_devices.empty()) {
        return 0; // nothing cached, no HIP call needed
    }
    int cur = 0;
    (void)hipGetDevice(&cur);
    hipError_t first = hipSuccess;
    for (auto& dv : g_devices) {
        DeviceCache& dc = dv.second;
        hipError_t e = hipSetDevice(dv.first);
        for (auto it = dc.entries.begin(); e == hipSuccess && it != dc.entries.end();) {
            Entry& ent = it->second;
            if (ent.busy) {
                ++it;
                continue;
            }
            if (ent.last_use != nullptr) {
                e = hipEventSynchronize(ent.last_use);
            }
            if (e == hipSuccess && ent.ptr != nullptr) {
                e = hipFreeAsync(ent.ptr, nullptr);
            }
            if (e != hipSuccess) {
                break;
            }
            if (ent.last_use != nullptr) {
                (void)hipEventDestroy(ent.last_use);
            }
            dc.bytes -= ent.bytes;
            it = dc.entries.erase(it);
        }
        if (e == hipSuccess) {
            e = hipDeviceSynchronize();
        }
        hipMemPool_t pool = nullptr;
        if (e == hipSuccess) {
            e = hipDeviceGetDefaultMemPool(&pool, dv.first);
        }
        if (e == hipSuccess) {
            e = hipMemPoolTrimTo(pool, 0);
        }
        if (e != hipSuccess && first == hipSuccess) {
            first = e;
        }
    }
    (void)hipSetDevice(cur);
    if (first != hipSuccess) {
        err = hip_err("scratch trim", first);
        return -1;
    }
    return 0;
}

int scratch_stats(int device, uint64_t& cached_bytes, int64_t& entries, int64_t& allocations) {
    std::lock_guard<std::mutex> lock(g_mu);
    auto it = g_devices.find(device);
    cached_bytes = 0;
    entries = 0;
    allocations = 0;
    if (it != g_devices.end()) {
        cached_bytes = it->second.bytes;
        for (const auto& kv : it->second.entries) {
            entries += kv.second.ptr != nullptr ? 1 : 0;
        }
        allocations = it->second.allocations;
    }
    return 0;
}

void graph_scratch_stats(int device, uint64_t& bytes, int64_t& blocks) {
    GraphBlocks& g = graph_blocks();
    std::lock_guard<std::mutex> lock(g.mu);
    const auto it = g.made.find(device);
    bytes = it != g.made.end() ? it->second.first : 0;
    blocks = it != g.made.end() ? it->second.second : 0;
}

} // namespace rdna_amd
