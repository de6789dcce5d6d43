// Per-GPU contexts, scratch workspace, device error word and host<->device
// copies of the B200 layer (see runtime.hpp).

#include "runtime.hpp"

#include <cuda.h>

#include <array>
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

void* nb2_device::scratch(size_t bytes) {
    bytes = (bytes + 255) & ~size_t(255);
    if (bytes <= workspace_bytes) {
        return workspace;
    }
    if (in_capture()) {
        nb2::fail(nb2::kStatusInvalid, "workspace must be sized before CUDA-graph capture");
    }
    nb2::check_cuda(cudaStreamSynchronize(stream), "cudaStreamSynchronize(workspace grow)");
    if (workspace != nullptr && callers_stream) {
        // a graph that the caller captured may still hold its address
        retired_split.push_back(workspace);
        workspace = nullptr;
        workspace_bytes = 0;
    }
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

int nb2_device::take_device_error() {
    int code = 0;
    nb2::check_cuda(cudaMemcpyAsync(&code, err_word, sizeof(int), cudaMemcpyDeviceToHost, stream),
                    "cudaMemcpyAsync(error word)");
    nb2::check_cuda(cudaStreamSynchronize(stream), "cudaStreamSynchronize");
    if (code != 0) {
        nb2::check_cuda(cudaMemsetAsync(err_word, 0, sizeof(int), stream), "cudaMemsetAsync(error word)");
        nb2::check_cuda(cudaStreamSynchronize(stream), "cudaStreamSynchronize");
    }
    return code;
}
