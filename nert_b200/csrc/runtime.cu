// Per-GPU contexts, scratch workspace, device error word and host<->device
// copies of the B200 layer (see runtime.hpp).

#include "runtime.hpp"

#include <cuda.h>

#include <algorithm>
#include <array>
#include <atomic>
#include <cstring>
#include <memory>

namespace nb2 {

namespace {
thread_local std::string g_last_error;
std::mutex g_devices_mu;
std::array<std::unique_ptr<nb2_device>, 64> g_devices;
} // namespace

void set_last_error(const std::string& msg) { g_last_error = msg; }
const char* last_error() { return g_last_error.c_str(); }

void fail(int code, const std::string& msg) { throw Error(code, msg); }

void check_cuda(cudaError_t e, const char* what) {
    if (e != cudaSuccess) {
        fail(kStatusCuda, std::string(what) + ": " + cudaGetErrorString(e));
    }
}

EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        check_cuda(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q),
                   "cudaGetDriverEntryPoint(cuTensorMapEncodeTiled)");
        if (p == nullptr || q != cudaDriverEntryPointSuccess) {
            fail(kStatusCuda, "cuTensorMapEncodeTiled is unavailable");
        }
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

EncodeIm2colFn encode_im2col() {
    static EncodeIm2colFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        check_cuda(cudaGetDriverEntryPoint("cuTensorMapEncodeIm2col", &p, cudaEnableDefault, &q),
                   "cudaGetDriverEntryPoint(cuTensorMapEncodeIm2col)");
        if (p == nullptr || q != cudaDriverEntryPointSuccess) {
            fail(kStatusCuda, "cuTensorMapEncodeIm2col is unavailable");
        }
        return reinterpret_cast<EncodeIm2colFn>(p);
    }();
    return fn;
}

namespace {

// A context of the GPU with its error word; the caller sets the stream.
std::unique_ptr<nb2_device> make_device(int ordinal) {
    int count = 0;
    check_cuda(cudaGetDeviceCount(&count), "cudaGetDeviceCount");
    if (ordinal >= count) {
        fail(kStatusInvalid, "no CUDA device " + std::to_string(ordinal));
    }
    cudaDeviceProp prop{};
    check_cuda(cudaGetDeviceProperties(&prop, ordinal), "cudaGetDeviceProperties");
    if (prop.major != 10) {
        fail(kStatusUnsupported, std::string("the B200 layer needs an sm_100 GPU, found ") + prop.name);
    }
    auto dev = std::make_unique<nb2_device>();
    dev->ordinal = ordinal;
    dev->num_sms = prop.multiProcessorCount;
    check_cuda(cudaSetDevice(ordinal), "cudaSetDevice");
    if (const char* env = std::getenv("NERT_B200_PRECISION")) {
        if (std::strcmp(env, "1xtf32") == 0 || std::strcmp(env, "1") == 0) {
            dev->precision = kPrec1xTF32;
        }
    }
    return dev;
}

void make_error_word(nb2_device* dev) {
    check_cuda(cudaMalloc(&dev->err_word, 256), "cudaMalloc(error word)");
    check_cuda(cudaMemsetAsync(dev->err_word, 0, 256, dev->stream), "cudaMemsetAsync(error word)");
    check_cuda(cudaStreamSynchronize(dev->stream), "cudaStreamSynchronize");
}

// Error words of the graphs that callers captured, one a GPU, made with its
// first context on a caller's stream.
struct GraphErrors {
    int* word = nullptr;
    std::atomic<bool> used{false}; // a graph holds it
};
std::array<GraphErrors, 64> g_graph_errors;

void make_graph_error_word(nb2_device* dev) {
    std::lock_guard<std::mutex> lock(g_devices_mu);
    GraphErrors& e = g_graph_errors[dev->ordinal];
    if (e.word == nullptr) {
        int* word = nullptr;
        check_cuda(cudaMalloc(&word, 256), "cudaMalloc(graph error word)");
        check_cuda(cudaMemsetAsync(word, 0, 256, dev->stream), "cudaMemsetAsync(graph error word)");
        check_cuda(cudaStreamSynchronize(dev->stream), "cudaStreamSynchronize");
        e.word = word;
    }
}

// Takes a word that other streams may be writing.
__global__ void take_word_kernel(int* word, int* to) { *to = atomicExch(word, 0); }

// Memory of graphs that callers capture: a block belongs to one graph, which
// gives it back when it and its executables are gone, and is then the next
// capture's. Blocks are never freed: the release runs on a thread of the
// driver's, where no CUDA call may be made.
struct GraphBlock {
    void* ptr = nullptr;
    size_t bytes = 0;
    std::atomic<bool> used{false};
};
std::mutex g_graph_mu;
std::array<std::vector<GraphBlock*>, 64>& graph_blocks() {
    static auto* blocks = new std::array<std::vector<GraphBlock*>, 64>; // outlives every release
    return *blocks;
}

void CUDART_CB release_graph_block(void* block) { static_cast<GraphBlock*>(block)->used = false; }

// At least `bytes` on the current GPU for the life of `graph`, during its capture.
void* graph_memory(int ordinal, cudaGraph_t graph, size_t bytes) {
    std::lock_guard<std::mutex> lock(g_graph_mu);
    auto& blocks = graph_blocks()[ordinal];
    GraphBlock* block = nullptr;
    for (GraphBlock* b : blocks) { // the smallest that is free and large enough
        if (!b->used && b->bytes >= bytes && (block == nullptr || b->bytes < block->bytes)) {
            block = b;
        }
    }
    if (block == nullptr) {
        auto fresh = std::make_unique<GraphBlock>();
        // an allocation is no work of the stream: it may be made during a capture by a thread that says so
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        check_cuda(cudaThreadExchangeStreamCaptureMode(&mode), "cudaThreadExchangeStreamCaptureMode");
        const cudaError_t e = cudaMalloc(&fresh->ptr, bytes);
        cudaThreadExchangeStreamCaptureMode(&mode);
        check_cuda(e, "cudaMalloc(graph workspace)");
        fresh->bytes = bytes;
        blocks.push_back(fresh.get());
        block = fresh.release();
    }
    cudaUserObject_t owner = nullptr;
    check_cuda(cudaUserObjectCreate(&owner, block, release_graph_block, 1, cudaUserObjectNoDestructorSync),
               "cudaUserObjectCreate");
    block->used = true;
    const cudaError_t e = cudaGraphRetainUserObject(graph, owner, 1, cudaGraphUserObjectMove);
    if (e != cudaSuccess) {
        cudaUserObjectRelease(owner, 1);
        check_cuda(e, "cudaGraphRetainUserObject");
    }
    return block->ptr;
}

} // namespace

nb2_device* device(int ordinal) {
    if (ordinal < 0 || ordinal >= 64) {
        fail(kStatusInvalid, "device ordinal out of range");
    }
    std::lock_guard<std::mutex> lock(g_devices_mu);
    if (!g_devices[ordinal]) {
        auto dev = make_device(ordinal);
        check_cuda(cudaStreamCreateWithFlags(&dev->stream, cudaStreamNonBlocking), "cudaStreamCreate");
        make_error_word(dev.get());
        g_devices[ordinal] = std::move(dev);
    }
    return g_devices[ordinal].get();
}

nb2_device* device_on_stream(int ordinal, cudaStream_t stream) {
    if (ordinal < 0 || ordinal >= 64) {
        fail(kStatusInvalid, "device ordinal out of range");
    }
    auto dev = make_device(ordinal);
    dev->callers_stream = true;
    dev->stream = stream;
    if (dev->in_capture()) {
        fail(kStatusInvalid, "a context must be made before its stream's CUDA-graph capture");
    }
    make_error_word(dev.get());
    make_graph_error_word(dev.get());
    return dev.release();
}

void release_device(nb2_device* dev) {
    if (!dev->callers_stream) {
        fail(kStatusInvalid, "only a context from nb2_device_on_stream is released");
    }
    dev->make_current();
    check_cuda(cudaStreamSynchronize(dev->stream), "cudaStreamSynchronize(release)");
    for (void* p : {static_cast<void*>(dev->err_word), dev->workspace, dev->split_ws,
                    static_cast<void*>(dev->ticket_ws)}) {
        check_cuda(cudaFree(p), "cudaFree(release)");
    }
    for (const auto* list : {&dev->retired_split, &dev->retired_tickets}) {
        for (void* p : *list) {
            check_cuda(cudaFree(p), "cudaFree(release)");
        }
    }
    if (dev->pinned != nullptr) {
        check_cuda(cudaFreeHost(dev->pinned), "cudaFreeHost(release)");
    }
    delete dev;
}

} // namespace nb2

nb2_device::nb2_device() : wait_bound(nb2::kDefaultWaitBoundCycles) {}

void nb2_device::make_current() const { nb2::check_cuda(cudaSetDevice(ordinal), "cudaSetDevice"); }

cudaGraph_t nb2_device::callers_graph() {
    if (!callers_stream) {
        return nullptr;
    }
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    cudaGraph_t graph = nullptr;
    if (cudaStreamGetCaptureInfo(stream, &st, &id, &graph) != cudaSuccess) {
        cudaGetLastError(); // the legacy stream while another stream captures
        return nullptr;
    }
    if (st != cudaStreamCaptureStatusActive) {
        return nullptr;
    }
    if (captured.id != id) {
        captured = Captured{};
        captured.id = id;
    }
    return graph;
}

void* nb2_device::scratch(size_t bytes) {
    bytes = (bytes + 255) & ~size_t(255);
    if (const cudaGraph_t graph = callers_graph()) {
        if (bytes > captured.workspace_bytes) {
            captured.workspace = nb2::graph_memory(ordinal, graph, bytes);
            captured.workspace_bytes = bytes;
        }
        return captured.workspace;
    }
    if (bytes <= workspace_bytes) {
        return workspace;
    }
    if (in_capture()) {
        nb2::fail(nb2::kStatusInvalid, "workspace must be sized before CUDA-graph capture");
    }
    nb2::check_cuda(cudaStreamSynchronize(stream), "cudaStreamSynchronize(workspace grow)");
    if (workspace != nullptr) {
        nb2::check_cuda(cudaFree(workspace), "cudaFree(workspace)");
        workspace = nullptr;
        workspace_bytes = 0;
    }
    const size_t grow = std::max(bytes, workspace_bytes * 2);
    nb2::check_cuda(cudaMalloc(&workspace, grow), "cudaMalloc(workspace)");
    workspace_bytes = grow;
    return workspace;
}

void* nb2_device::split_scratch(size_t bytes) {
    bytes = (bytes + 255) & ~size_t(255);
    if (no_grow) {
        return nullptr; // a no-allocation call never depends on this shared buffer
    }
    if (const cudaGraph_t graph = callers_graph()) {
        if (bytes > captured.split_ws_bytes) {
            captured.split_ws = nb2::graph_memory(ordinal, graph, bytes);
            captured.split_ws_bytes = bytes;
        }
        return captured.split_ws;
    }
    if (bytes <= split_ws_bytes) {
        return split_ws;
    }
    if (in_capture()) {
        return nullptr; // the caller then runs the contraction unsplit
    }
    const size_t grow = std::max(bytes, split_ws_bytes * 2);
    void* fresh = nullptr;
    nb2::check_cuda(cudaMalloc(&fresh, grow), "cudaMalloc(split workspace)");
    if (split_ws != nullptr) {
        retired_split.push_back(split_ws);
    }
    split_ws = fresh;
    split_ws_bytes = grow;
    return split_ws;
}

uint32_t* nb2_device::tickets(size_t n) {
    if (const cudaGraph_t graph = callers_graph()) {
        if (n > captured.ticket_count) {
            const size_t count = std::max<size_t>(n, 4096);
            captured.ticket_ws = static_cast<uint32_t*>(nb2::graph_memory(ordinal, graph, count * sizeof(uint32_t)));
            captured.ticket_count = count;
            // a node of the graph: each replay begins with zeros
            nb2::check_cuda(cudaMemsetAsync(captured.ticket_ws, 0, count * sizeof(uint32_t), stream),
                            "cudaMemsetAsync(graph tickets)");
        }
        return captured.ticket_ws;
    }
    if (n <= ticket_count) {
        return ticket_ws;
    }
    if (in_capture()) {
        nb2::fail(nb2::kStatusInvalid, "workspace must be sized before CUDA-graph capture");
    }
    const size_t grow = std::max(n, std::max<size_t>(4096, ticket_count * 2));
    uint32_t* fresh = nullptr;
    nb2::check_cuda(cudaMalloc(&fresh, grow * sizeof(uint32_t)), "cudaMalloc(tickets)");
    nb2::check_cuda(cudaMemsetAsync(fresh, 0, grow * sizeof(uint32_t), stream), "cudaMemsetAsync(tickets)");
    if (ticket_ws != nullptr) {
        retired_tickets.push_back(ticket_ws);
    }
    ticket_ws = fresh;
    ticket_count = grow;
    return ticket_ws;
}

bool nb2_device::in_capture() const {
    if (capturing) {
        return true;
    }
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream, &st) != cudaSuccess) {
        cudaGetLastError(); // the legacy stream while another stream captures
        return true;
    }
    return st != cudaStreamCaptureStatusNone;
}

int* nb2_device::error_word() {
    if (callers_graph() == nullptr) {
        return err_word;
    }
    nb2::GraphErrors& e = nb2::g_graph_errors[ordinal];
    e.used = true;
    return e.word;
}

int nb2_device::take_device_error() {
    // two threads that wait for one context take turns: each reads the words, then clears them
    std::lock_guard<std::mutex> lock(mu);
    int codes[2] = {0, 0}; // this context's, replayed graphs'
    const nb2::GraphErrors& graphs = nb2::g_graph_errors[ordinal];
    const bool with_graphs = callers_stream && graphs.used;
    if (with_graphs) {
        nb2::take_word_kernel<<<1, 1, 0, stream>>>(graphs.word, err_word + 1);
        nb2::check_cuda(cudaGetLastError(), "error word launch");
    }
    nb2::check_cuda(cudaMemcpyAsync(codes, err_word, (with_graphs ? 2 : 1) * sizeof(int), cudaMemcpyDeviceToHost, stream),
                    "cudaMemcpyAsync(error word)");
    nb2::check_cuda(cudaStreamSynchronize(stream), "cudaStreamSynchronize");
    if (codes[0] != 0) {
        nb2::check_cuda(cudaMemsetAsync(err_word, 0, sizeof(int), stream), "cudaMemsetAsync(error word)");
        nb2::check_cuda(cudaStreamSynchronize(stream), "cudaStreamSynchronize");
    }
    return codes[0] != 0 ? codes[0] : codes[1];
}
