// Host-side checks shared by the entry points on DEVICE tensors (residual_norm.hip, grad_clip.hip).
#pragma once
#include "sr_internal.h"

namespace srh {

// `device` made current for the length of a call; the caller's current device comes back on every path.
struct OnDevice {
    int prev = -1;
    int enter(int device) {
        int ndev = 0, cur = -1;
        if (hipGetDeviceCount(&ndev) != hipSuccess || ndev == 0)
            return fail(nullptr, SR_ERR_HIP, "no HIP device available; libsr_hip has no CPU fallback");
        if (device < 0 || device >= ndev) return fail(nullptr, SR_ERR_ARG, "device %d out of range", device);
        if (hipGetDevice(&cur) != hipSuccess) return fail(nullptr, SR_ERR_HIP, "hipGetDevice failed");
        if (cur != device) {
            if (hipSetDevice(device) != hipSuccess) return fail(nullptr, SR_ERR_HIP, "hipSetDevice failed");
            prev = cur;
        }
        return SR_OK;
    }
    ~OnDevice() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

// bytes of one element of enum sr_type; 0: no such type
inline int type_bytes(int type) { return type == SR_T_F32 ? 4 : (type == SR_T_BF16 || type == SR_T_F16) ? 2 : 0; }

// `rows` rows of `width` bytes, `pitch` bytes apart (width <= pitch where rows > 1)
struct Region {
    const char* p = nullptr;
    int64_t rows = 0, pitch = 0, width = 0;
    bool empty() const { return !p || rows == 0 || width == 0; }
    const char* end() const { return p + (rows - 1) * pitch + width; }
};

inline bool disjoint(const Region& a, const Region& b) {
    if (a.empty() || b.empty() || a.end() <= b.p || b.end() <= a.p) return true;
    if (a.pitch != b.pitch || a.rows < 2 || b.rows < 2) return false;
    // column blocks of one wider matrix
    const int64_t d = ((b.p - a.p) % a.pitch + a.pitch) % a.pitch;
    return d >= a.width && d + b.width <= a.pitch;
}

inline bool same(const Region& a, const Region& b) {
    return a.p == b.p && a.rows == b.rows && a.width == b.width && (a.pitch == b.pitch || a.rows < 2);
}

}  // namespace srh
