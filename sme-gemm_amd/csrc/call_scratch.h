// Scratch that one device-pointer call holds while it enqueues its launches.
//
// An eager call leases its stream's buffer (lease_pool.h): calls of several host
// threads on one stream stay apart, and an outgrown buffer is given back. A call on
// a stream that is being captured takes a buffer of that capture's own, which is kept
// until the process ends, as the graph may be launched at any time: no two graphs,
// and no graph and eager call, share one. Within a capture the calls of one stream
// are ordered by that stream and share a buffer; a branch captured from another
// stream has its own. A caller that brings scratch of its own uses that, and says when it
// ends: HIP tells the library nothing when a graph does (a user object that the captured
// graph retains is not released with the instantiated one).
#pragma once

#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <utility>

#include "api_internal.h"
#include "lease_pool.h"
#include "scratch_pool.h"

namespace smg {

struct CallAlloc {
    // allocating (or freeing) is an error in a thread of the default capture mode
    // while a stream is captured
    struct Relaxed {
        hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
        Relaxed() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
        ~Relaxed() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
    };
    void *acquire(int, size_t bytes) {  // (the caller has made the device current)
        Relaxed r;
        void *p = nullptr;
        return device_malloc(&p, bytes) == hipSuccess ? p : nullptr;
    }
    void release(int, void *p) {
        Relaxed r;
        (void)hipFree(p);  // waits for the device
    }
};

// A caller's scratch: on the call's device, at a multiple of 256 bytes.
struct OwnScratch {
    void *buf;
    size_t bytes;
};

class CallScratch {
public:
    // `bytes` (0: none) for a call on (device, stream), the device being current; the
    // caller's own, if there is one.
    CallScratch(int device, void *stream, size_t bytes, const OwnScratch *mine) {
        if (mine) {
            buf_ = mine->buf;
            if (bytes > mine->bytes || (bytes && (!buf_ || (uintptr_t)buf_ % 256))) error_ = hipErrorInvalidValue;
            return;
        }
        if (bytes == 0) return;
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        unsigned long long id = 0;
        error_ = hipStreamGetCaptureInfo((hipStream_t)stream, &st, &id);
        if (error_ != hipSuccess) {  // (the null stream beside a blocking one's capture)
            (void)hipGetLastError();
            return;
        }
        // each thread's own stream has one handle
        static thread_local char own;
        const void *key = stream == (void *)hipStreamPerThread ? (const void *)&own : stream;
        if (st == hipStreamCaptureStatusNone) {
            static LeasePool<CallAlloc> *pool = new LeasePool<CallAlloc>(32, (size_t)64 << 30);  // never destroyed
            lease_ = pool->take(device, key, bytes);
            buf_ = lease_.buf();
        } else if (st == hipStreamCaptureStatusActive) {
            static std::mutex *mu = new std::mutex;
            static auto *keys = new std::map<std::pair<unsigned long long, const void *>, std::unique_ptr<char>>;
            static ScratchPool<CallAlloc> *pool = new ScratchPool<CallAlloc>();
            std::lock_guard<std::mutex> lk(*mu);
            std::unique_ptr<char> &k = (*keys)[{id, key}];
            if (!k) k.reset(new char);
            buf_ = pool->get(device, k.get(), bytes);
        } else {
            error_ = hipErrorStreamCaptureInvalidated;
            return;
        }
        if (!buf_) error_ = hipErrorOutOfMemory;
    }
    // SMG_OK, or the failure, reported for `call`.
    int check(const char *call) const {
        if (error_ == hipSuccess) return SMG_OK;
        if (error_ == hipErrorInvalidValue)
            return report(SMG_EINVAL, (std::string(call) + ": scratch too small, or not at a multiple of 256 bytes").c_str());
        if (error_ == hipErrorOutOfMemory) return report(SMG_ENOMEM, (std::string(call) + ": scratch hipMalloc").c_str());
        return report_hip(SMG_EHIP, call, error_);
    }
    void *buf() const { return buf_; }

private:
    LeasePool<CallAlloc>::Lease lease_;
    void *buf_ = nullptr;
    hipError_t error_ = hipSuccess;
};

// Makes a device current for a scope.
class DeviceScope {
public:
    explicit DeviceScope(int device) {
        if (hipGetDevice(&old_) != hipSuccess) old_ = -1;
        e_ = old_ == device ? hipSuccess : hipSetDevice(device);
        if (old_ == device) old_ = -1;
    }
    ~DeviceScope() {
        if (old_ >= 0) (void)hipSetDevice(old_);
    }
    hipError_t error() const { return e_; }

private:
    int old_ = -1;
    hipError_t e_ = hipSuccess;
};

}  // namespace smg
