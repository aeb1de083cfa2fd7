// Tensor arguments of the decoder blocks' entry points (blocks.cpp, block_cache.cpp): what a call holds, and its activations as rows.
#pragma once

#include "blocks.hpp"

namespace cg {

// The consumed references of a block's tensor arguments, and the temporaries made from them.
struct Held {
    std::vector<cg_tensor *> t;
    ~Held() {
        for (cg_tensor *x : t) release(x);
    }
    cg_tensor *add(cg_tensor *x) {
        t.push_back(x);
        return x;
    }
};

// Pool memory for the duration of a call (stream-ordered: whoever gets it next queues behind this call's kernels).
struct Scratch {
    explicit Scratch(cg_backend *b) : be(b) {}
    ~Scratch() {
        for (auto &a : mem) be->pool.free(a.first, a.second);
    }
    int get(size_t bytes, void **p) {
        size_t cls;
        int rc = be->pool.alloc(bytes ? bytes : 4, p, &cls);
        if (!rc) mem.emplace_back(*p, cls);
        return rc;
    }
    cg_backend *be;
    std::vector<std::pair<void *, size_t>> mem;
};

inline int check_float(const cg_tensor *t, const char *what) {
    return is_f(t->dt) ? CG_OK : fail(CG_ERR_DTYPE, "%s: expected a floating-point tensor", what);
}

// t as rows of its last axis, `rows` x `features`, every row with unit stride and one distance from row to row.
inline int rows_of(cg_backend *be, Held &h, cg_tensor *t, int64_t rows, int64_t features, Rows *out, const char *what) {
    if (int rc = check_float(t, what)) return rc;
    if (t->rank < 1 || t->dims[t->rank - 1] != features || numel(t) != rows * features)
        return fail(CG_ERR_SHAPE, "%s: expected %lld rows of %lld", what, (long long)rows, (long long)features);
    if (int rc = ensure_concrete(t)) return rc;
    bool regular = !t->uniform && (features == 1 || t->strides[t->rank - 1] == 1);
    int64_t pitch = features, run = -1; // run: distance after which the next outer axis has to continue
    for (int d = t->rank - 2; d >= 0 && regular; d--) {
        if (t->dims[d] == 1) continue;
        if (run < 0) {
            pitch = t->strides[d];
            run = pitch;
        } else if (t->strides[d] != run) {
            regular = false;
        }
        run *= t->dims[d];
    }
    if (!regular) {
        cg_tensor *m = nullptr;
        if (int rc = materialize(be, t, &m)) return rc;
        h.add(m);
        t = m;
        pitch = features;
    }
    const void *p;
    if (int rc = device_ptr(t, &p)) return rc;
    out->p = static_cast<const float *>(p);
    out->pitch = pitch;
    return CG_OK;
}

inline int check_sizes(int64_t rows, int64_t a, int64_t b) {
    return rows < (1ll << 31) && a < (1ll << 31) && b < (1ll << 31) ? CG_OK : fail(CG_ERR_UNSUPPORTED, "block: an extent exceeds 2^31");
}

} // namespace cg

#define CG_ENTER_BLOCK(b)                                                                             \
    if (!(b)) return fail(CG_ERR_ARG, "null argument");                                               \
    if ((b)->owner_gone) return fail(CG_ERR_ARG, "backend used after cg_backend_destroy");            \
    CG_HIP(hipSetDevice((b)->device));                                                                \
    if (int flush_rc = flush_deferred(b)) return flush_rc
