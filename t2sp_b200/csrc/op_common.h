// Argument checks and call plumbing shared by the translation units that hold the operator entry points: the
// halide_error_* reporters, the checks in the order the generated host code performs them, the views a call holds
// and its synchronous end.
#pragma once
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <initializer_list>
#include <string>

#include "host_rt.h"

extern "C" {
int halide_error_bad_type(void*, const char*, uint32_t, uint32_t);
int halide_error_bad_dimensions(void*, const char*, int32_t, int32_t);
int halide_error_access_out_of_bounds(void*, const char*, int, int, int, int, int);
int halide_error_buffer_allocation_too_large(void*, const char*, uint64_t, uint64_t);
int halide_error_buffer_extents_negative(void*, const char*, int, int);
int halide_error_buffer_extents_too_large(void*, const char*, int64_t, int64_t);
int halide_error_constraint_violated(void*, const char*, int, const char*, int);
int halide_error_buffer_argument_is_null(void*, const char*);
int halide_error_host_is_null(void*, const char*);
}

namespace t2sp {
cudaEvent_t rt_event(int which);

namespace {

constexpr uint32_t type_word(int code, int bits) { return uint32_t(code) | (uint32_t(bits) << 8) | (1u << 16); }
constexpr uint32_t kF32 = type_word(2, 32), kBF16 = type_word(4, 16), kF16 = type_word(2, 16), kI8 = type_word(0, 8),
                   kI32 = type_word(0, 32), kU8 = type_word(1, 8);

uint32_t buf_type_word(const halide_buffer_t* b) {
    uint32_t w;
    memcpy(&w, &b->type, 4);
    return w;
}

struct Arg {
    halide_buffer_t* b;
    const char* name;   // "A"
    bool is_output;
    int dims;
    std::string role() const { return std::string(is_output ? "Output buffer " : "Input buffer ") + name; }
};

// Fills a bounds-query buffer with a dense shape of the given extents.
void fill_query(halide_buffer_t* b, uint32_t tword, int dims, const int* ext) {
    memcpy(&b->type, &tword, 4);
    b->dimensions = dims;
    int64_t stride = 1;
    for (int d = 0; d < dims; ++d) {
        b->dim[d].min = 0;
        b->dim[d].extent = ext[d];
        b->dim[d].stride = static_cast<int32_t>(stride);
        b->dim[d].flags = 0;
        stride *= ext[d];
    }
}

int check_null(const Arg* args, int n) {
    // the generated code tests the output first, then the inputs last to first
    for (int i = n - 1; i >= 0; --i)
        if (!args[i].b) return halide_error_buffer_argument_is_null(nullptr, args[i].name);
    return 0;
}

int check_type_dims(const Arg& a, uint32_t want) {
    if (buf_type_word(a.b) != want) return halide_error_bad_type(nullptr, a.role().c_str(), buf_type_word(a.b), want);
    if (a.b->dimensions != a.dims)
        return halide_error_bad_dimensions(nullptr, a.role().c_str(), a.b->dimensions, a.dims);
    return 0;
}

int check_extents_nonneg(const Arg& a) {
    for (int d = 0; d < a.b->dimensions; ++d)
        if (a.b->dim[d].extent < 0)
            return halide_error_buffer_extents_negative(nullptr, a.role().c_str(), d, a.b->dim[d].extent);
    return 0;
}

// The buffer must cover [0, need-1] in dimension d.
int check_covers(const Arg& a, int d, int need) {
    const int mn = a.b->dim[d].min, mx = mn + a.b->dim[d].extent - 1;
    if (mn > 0 || mx < need - 1)
        return halide_error_access_out_of_bounds(nullptr, a.role().c_str(), d, 0, need - 1, mn, mx);
    return 0;
}

int check_stride0(const Arg& a) {
    if (a.b->dim[0].stride != 1) {
        std::string v = std::string(a.name) + ".stride.0";
        return halide_error_constraint_violated(nullptr, v.c_str(), a.b->dim[0].stride, "1", 1);
    }
    return 0;
}

int check_sizes(const Arg& a) {
    const int64_t span = buf_elems_span(a.b);
    const int64_t bytes = span * ((a.b->type.bits + 7) / 8);
    // The reference caps a buffer at 2^31-1 bytes because its indices are 32-bit
    // (syrk-interface.cpp:368-432); here indices are 64-bit and the cap is the 2^31-1 limit
    // of Halide's int32 extents and strides themselves.
    int64_t prod = 1;
    for (int d = 0; d < a.b->dimensions; ++d) {
        prod *= std::max(a.b->dim[d].extent, 1);
        if (prod > (int64_t(1) << 40))
            return halide_error_buffer_extents_too_large(nullptr, a.name, prod, int64_t(1) << 40);
    }
    if (bytes > (int64_t(1) << 40))
        return halide_error_buffer_allocation_too_large(nullptr, a.name, bytes, uint64_t(1) << 40);
    return 0;
}

int check_host(const Arg& a) {
    if (!a.b->host && !buf_on_our_device(a.b)) return halide_error_host_is_null(nullptr, a.role().c_str());
    return 0;
}

int constraint(const char* var, int val, const char* want_name, int want) {
    return halide_error_constraint_violated(nullptr, var, val, want_name, want);
}

// Offset (elements) from the buffer's first stored element to coordinate 0 in every dimension.
int64_t origin_offset(const halide_buffer_t* b) {
    int64_t off = 0;
    for (int d = 0; d < b->dimensions; ++d) off -= int64_t(b->dim[d].min) * b->dim[d].stride;
    return off;
}

bool tma_ok(const void* base, std::initializer_list<int64_t> strides_bytes) {
    if (reinterpret_cast<uintptr_t>(base) & 15) return false;
    for (int64_t s : strides_bytes)
        if (s <= 0 || (s & 15)) return false;
    return true;
}

int tma_unsupported(const char* name) {
    fprintf(stderr,
            "t2sp_b200: buffer %s cannot be read by TMA in place (base address and every outer stride must be "
            "16-byte aligned)\n",
            name);
    return halide_error_code_constraint_violated;
}

int finish_call(const char* who, const char* kernel_name, bool sync_after) {
    if (!sync_after) return 0;
    int rc = rt_check_status(who);
    if (rc) return rc;
    float ms = 0.f;
    if (cudaEventElapsedTime(&ms, rt_event(0), rt_event(1)) == cudaSuccess) {
        tls().last_kernel_ns = double(ms) * 1e6;
        rt_write_exec_time(kernel_name, tls().last_kernel_ns);
    }
    if (rt_env().log) fprintf(stderr, "t2sp_b200: %s: kernels %.1f us\n", who, tls().last_kernel_ns * 1e-3);
    return 0;
}

bool all_resident(std::initializer_list<const halide_buffer_t*> bufs) {
    for (auto* b : bufs)
        if (!buf_on_our_device(b) || ((b->flags & 1u) && b->host)) return false;
    return true;
}

struct Views {
    DeviceView v[8];
    int n = 0;
    ~Views() {
        for (int i = 0; i < n; ++i) rt_drop_view(&v[i]);
    }
};

// Every coordinate of the buffer starts at 0 (the extents alone then say what is read).
int check_min0(const Arg& a) {
    for (int d = 0; d < a.b->dimensions; ++d)
        if (int e = check_covers(a, d, a.b->dim[d].extent)) return e;
    return 0;
}

// Outer strides that address memory forwards; for an output also without two coordinates on one element.
int check_strides(const Arg& a) {
    int64_t reach = 1;   // elements from the first to behind the last that the dimensions so far address, in the order of their strides
    int order[8], n = 0;
    for (int d = 0; d < a.b->dimensions; ++d)
        if (a.b->dim[d].extent == 0) return 0;
    for (int d = 0; d < a.b->dimensions && n < 8; ++d)
        if (a.b->dim[d].extent > 1) order[n++] = d;
    std::sort(order, order + n, [&](int x, int y) { return a.b->dim[x].stride < a.b->dim[y].stride; });
    for (int i = 0; i < n; ++i) {
        const int64_t stride = a.b->dim[order[i]].stride;
        if (stride <= 0 || (a.is_output && stride < reach)) {
            const std::string v = std::string(a.name) + ".stride." + std::to_string(order[i]);
            return constraint(v.c_str(), a.b->dim[order[i]].stride, a.is_output ? "at least the elements it strides over" : "positive",
                              static_cast<int>(std::min<int64_t>(reach, 0x7fffffff)));
        }
        reach += stride * (a.b->dim[order[i]].extent - 1);
    }
    return 0;
}

// The kernels of the entries with ragged shapes count in 32 bits and add a tile's length to an extent.
int check_extent_limit(const Arg& a) {
    for (int d = 0; d < a.b->dimensions; ++d)
        if (a.b->dim[d].extent > (1 << 30))
            return halide_error_buffer_extents_too_large(nullptr, a.name, a.b->dim[d].extent, int64_t(1) << 30);
    return 0;
}

// The buffers of a bounds query that say something: their extents are ones that a call takes.
int check_query_known(const Arg* args, int n) {
    for (int i = 0; i < n; ++i) {
        if (!args[i].b || buf_is_bounds_query(args[i].b)) continue;
        if (int e = check_extents_nonneg(args[i])) return e;
        if (int e = check_extent_limit(args[i])) return e;
    }
    return 0;
}

// A device address is a multiple of the element's size (the kernels that take any 16-bit alignment need at least that).
int check_device_address(const Arg& a) {
    const int bytes = (a.b->type.bits + 7) / 8, off = static_cast<int>(a.b->device % uint64_t(bytes));
    if (!buf_on_our_device(a.b) || off == 0) return 0;
    return constraint((std::string(a.name) + ".device").c_str(), off, "a multiple of the element's size", bytes);
}

// A call whose stream is being captured into a graph can neither wait for its kernels nor take scratch memory that
// the graph would go on using after the call has handed it back.
int check_capture(const char* who, bool waits, bool scratch) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(rt_stream(), &st) != cudaSuccess) { cudaGetLastError(); return 0; }
    if (st == cudaStreamCaptureStatusNone || (!waits && !scratch)) return 0;
    fprintf(stderr, "t2sp_b200: %s: the stream is being captured, and this call %s\n", who,
            waits ? "would wait for it (use device-resident buffers and t2sp_b200_set_async)"
                  : "needs scratch memory (give operands with a 16-byte aligned base and strides)");
    return halide_error_code_constraint_violated;
}

// An output that the call writes only in part starts from the caller's values: a device copy of host memory, and a device
// allocation whose host side is the newer one.
int preload_output(halide_buffer_t* b, DeviceView* v) {
    if (v->preloaded || v->bytes == 0) return 0;
    if (v->borrowed && !((b->flags & 1u) && b->host)) return 0;
    const bool ok = v->borrowed ? rt_move_buffer(b, false)
                                : cudaMemcpyAsync(v->ptr, b->host, v->bytes, cudaMemcpyHostToDevice, rt_stream()) == cudaSuccess;
    if (!ok) {
        cudaGetLastError();
        return halide_error_code_copy_to_device_failed;
    }
    return 0;
}

}  // namespace
}  // namespace t2sp
