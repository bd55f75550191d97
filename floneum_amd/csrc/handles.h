// What the library's opaque handles hold, for the C-ABI files.
#pragma once
#include <atomic>

#include "common.h"

struct fhip_device {
    int ordinal;
    hipDeviceProp_t prop;
    void *scratch_ptr;  // this device's address of `scratch`
    // Sources of the per-call marks of masked prefill calls (AttnParams::bad_tag) and of decode calls (dec_tag): the state a
    // device handle changes after its creation.
    std::atomic<uint32_t> next_tag;
    std::atomic<uint64_t> next_mark;
    // The fused split-KV merge needs workgroups L of a one-dimensional launch with the same L % 8 to share an XCD (and
    // with it an L2).  Probed once per handle.  `trip` is a word of pinned host memory the decode kernels set when the
    // workgroups of a unit find themselves on different XCDs all the same: the next decode call then fails once and the
    // form stays off for the handle.
    std::atomic<bool> xcd_grouped;
    int32_t *trip_host, *trip_dev;
};

struct fhip_stream {
    fhip_device *dev;
    hipStream_t s;
};
struct fhip_event {
    fhip_device *dev;
    hipEvent_t e;
};
struct fhip_graph {
    fhip_device *dev;
    hipGraph_t graph;
    hipGraphExec_t exec;
};
