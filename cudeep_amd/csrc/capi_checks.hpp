// Argument checks that the extern "C" files of the operators beside the reference's share: all
// run on the host before any launch, and say what is wrong through cdx_last_error().
#pragma once

#include <string>

#include "cdx_internal.hpp"

namespace cdx {
namespace checks {

constexpr int64_t kMaxDim = (int64_t)1 << 40;

inline int bad(const char* fn, const char* what) {
    return set_error(CDX_ERR_INVALID_ARG, std::string(fn) + ": " + what);
}

inline bool bad_dim(int64_t d) { return d < 0 || d > kMaxDim; }

// Every flat index (bytes included) fits in 64 bits with room to spare.
inline bool too_large(int64_t rows, int64_t ld) {
    return (long double)rows * (long double)ld > (long double)((int64_t)1 << 58);
}

inline bool float_dtype(int d) { return d == CDX_DTYPE_F32 || d == CDX_DTYPE_F16 || d == CDX_DTYPE_BF16; }
inline bool gemm_epilogue(int e) { return e >= CDX_EPI_NONE && e <= CDX_EPI_SIGMOID; }

// A row-major matrix argument; empty ones may be NULL.
inline int check_matrix(const char* fn, const char* name, const void* p, int64_t ld, int64_t rows,
                 int64_t cols) {
    if (ld < cols) return bad(fn, (std::string(name) + ": leading dimension too small").c_str());
    if (too_large(rows, ld)) return bad(fn, (std::string(name) + ": too large").c_str());
    if (rows > 0 && cols > 0 && !p) return bad(fn, (std::string(name) + " is NULL").c_str());
    return CDX_OK;
}

// A checked row-major matrix as the bytes of its rows.
struct Span {
    uintptr_t at; int64_t pitch, width, rows;
    Span(const void* p, int64_t ld, int64_t rows_, int64_t cols, int dtype)
        : at((uintptr_t)p), pitch(ld * size(dtype)), width(cols * size(dtype)), rows(rows_) {}
    static int64_t size(int dtype) { return dtype == CDX_DTYPE_F32 ? 4 : 2; }
    uintptr_t end() const { return at + (uintptr_t)((rows - 1) * pitch + width); }
    bool same(const Span& o) const { return at == o.at && (pitch == o.pitch || rows == 1); }
};

// Whether two of them share a byte.  Columns of one wider matrix that lie beside each other do not;
// rows of different pitches that mesh are taken to.
inline bool overlap(const Span& a, const Span& b) {
    if (a.rows == 0 || a.width == 0 || b.rows == 0 || b.width == 0) return false;
    if (a.end() <= b.at || b.end() <= a.at) return false;
    if (a.pitch != b.pitch) return true;
    const int64_t off = b.at >= a.at ? (int64_t)((b.at - a.at) % (uintptr_t)a.pitch)
                                     : a.pitch - 1 - (int64_t)((a.at - b.at - 1) % (uintptr_t)a.pitch);
    return !(off >= a.width && off + b.width <= a.pitch);
}

// A row operator's result: its input's own place, or apart from it (workgroups take rows in any order).
inline int check_in_place(const char* fn, const char* what, const Span& out, const Span& in) {
    if (out.same(in) || !overlap(out, in)) return CDX_OK;
    return bad(fn, (std::string(what) + " overlap without being the same").c_str());
}

struct NamedSpan { const char* name; Span at; };

// A call's results must share nothing with each other, nor with what is read while they are written.
template <size_t W, size_t R>
inline int check_results(const char* fn, const NamedSpan (&writes)[W], const NamedSpan (&reads)[R]) {
    auto apart = [&](const NamedSpan& a, const NamedSpan& b) {
        return overlap(a.at, b.at) ? bad(fn, (std::string(a.name) + " and " + b.name + " overlap").c_str()) : (int)CDX_OK;
    };
    for (size_t i = 0; i < W; ++i) {
        for (const NamedSpan& r : reads)
            if (const int st = apart(writes[i], r)) return st;
        for (size_t j = 0; j < i; ++j)
            if (const int st = apart(writes[i], writes[j])) return st;
    }
    return CDX_OK;
}

// Scratch that holds 16-byte pieces.
inline int check_workspace(const char* fn, const void* ws) {
    return (uintptr_t)ws % 16 ? bad(fn, "workspace must be 16-byte aligned") : (int)CDX_OK;
}

// Runs f(scratch) with the caller's workspace or stream-ordered memory.
template <class F>
inline int with_workspace(const char* fn, size_t need, void* ws, size_t ws_bytes, hipStream_t stream, F f) {
    if (need == 0) return f(static_cast<void*>(nullptr));
    if (ws) {
        if (ws_bytes < need)
            return set_error(CDX_ERR_WORKSPACE, std::string(fn) + ": workspace too small");
        return f(ws);
    }
    void* p = nullptr;
    int st = cdx::stream_alloc(&p, need, stream, fn);
    if (st) return st;
    st = f(p);
    const int st2 = cdx::stream_free(p, stream, fn);
    return st ? st : st2;
}

}  // namespace checks
}  // namespace cdx
