// Helpers shared by the entry points of tree attention, page copies and beam selection.
#pragma once

#include <cstdint>
#include <exception>

#include "ctx.hpp"

namespace mlcb {

// Runs the body of a C entry point; an exception (host memory that ran out) becomes a status.
template <typename F>
int no_throw(mlc_ctx* ctx, F&& body) {
    try {
        return body();
    } catch (const std::exception&) {
        try {
            if (ctx) ctx->last_error = "out of host memory";
        } catch (...) {
        }
        return MLC_ERR_OOM;
    }
}

// Device scratch of one kind of launch. It grows by adding a larger buffer; the smaller ones stay until the context
// goes, so that a graph captured with one of them can still be replayed. Launches of one context run in stream order,
// which is what lets them share it. Zero-filled when allocated.
int ensure_op_scratch(mlc_ctx* ctx, OpScratch& s, size_t bytes, const char* what);

// Notes that a launch enqueued just now writes into these pools: the decode launch enqueued next must not fetch
// from them before everything in front of it has finished.
void note_pool_writes(mlc_ctx* ctx, void* const* pools, size_t n_pools);

inline bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + b_bytes && y < x + a_bytes;
}
inline bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Launch as a programmatic dependent of the kernel in front: the kernel waits (griddepcontrol.wait) before it touches
// anything that another kernel reads or writes.
template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(mlc_ctx* ctx, void (*kernel)(KArgs...), dim3 grid, unsigned block, size_t smem, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

}  // namespace mlcb
