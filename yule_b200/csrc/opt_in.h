// opt_in.h — what kernels have been opted in to, by kernel and device.  No CUDA in it.
#pragma once

#include <cstddef>
#include <map>
#include <mutex>
#include <new>
#include <utility>

namespace yule {

// Every kernel of every device has an entry that is never given up: who asked for less later would take away what a larger call, on its way to its launch, has got.
class OptIns {
public:
    // `ask_smem(bytes)` and `ask_clusters()`, which make the calls and return 0, where this kernel has not got as much yet; what they return else, or `no_memory`.
    template <typename Smem, typename Clusters, typename E>
    E take(const void *kernel, int device, size_t smem, bool large_clusters, Smem ask_smem, Clusters ask_clusters, E no_memory) {
        std::lock_guard<std::mutex> lock(mu);
        Got *got;
        try {
            got = &all[{kernel, device}];
        } catch (const std::bad_alloc &) {
            return no_memory;
        }
        if (smem > got->smem) {
            if (const E e = ask_smem(smem); e != E{}) return e;
            got->smem = smem;
        }
        if (large_clusters && !got->large_clusters) {
            if (const E e = ask_clusters(); e != E{}) return e;
            got->large_clusters = true;
        }
        return E{};
    }

private:
    struct Got {
        size_t smem = 0;
        bool large_clusters = false;
    };
    std::map<std::pair<const void *, int>, Got> all;
    std::mutex mu;
};

}  // namespace yule
