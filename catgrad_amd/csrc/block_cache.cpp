// Entry points of rotary positions and the 8-bit key / value cache (their section of include/catgrad_hip.h), on tensors of a
// backend and on a caller's own device memory: argument checks, then the same kernels.
#include "block_cache.hpp"

#include "block_args.hpp"

#include <algorithm>
#include <cmath>
#include <exception>

namespace cg {
namespace {

constexpr uint64_t kMostPosition = 1ull << 40;
constexpr uint32_t kMostTokens = (1u << 24) - 1; // of a call: a workgroup each, and fewer than 2^32 threads of a launch

bool cache_dim(size_t n) { return n >= 16 && n <= 256 && n % 16 == 0; }
int block_log2(size_t n) { return n == 16 ? 4 : n == 32 ? 5 : n == 64 ? 6 : n == 128 ? 7 : -1; }
bool at16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_batch(size_t sequences, size_t tokens, uint64_t position, const char *what) {
    if (sequences > kMostTokens || tokens > kMostTokens || sequences * tokens > kMostTokens) return fail(CG_ERR_UNSUPPORTED, "%s: 2^24 tokens or more", what);
    if (position > kMostPosition) return fail(CG_ERR_RANGE, "%s: a position beyond 2^40", what);
    return CG_OK;
}

int check_rotation(size_t heads, size_t kv_heads, size_t dim, size_t rot, const char *what) {
    if (heads < 1 || dim < 2 || heads > 4096 || kv_heads > 4096 || dim > 4096) return fail(CG_ERR_ARG, "%s: bad head counts or sizes", what);
    if (rot < 2 || rot % 2 || rot > dim || rot > 512) return fail(CG_ERR_ARG, "%s: an even number of values up to 512 of a head is turned", what);
    return CG_OK;
}

// Sizes of a cache and of what is done with it.
int check_cache(size_t sequences, size_t tokens, size_t kv_heads, size_t dim, size_t vdim, size_t capacity, size_t block, const char *what) {
    if (!cache_dim(dim) || !cache_dim(vdim)) return fail(CG_ERR_UNSUPPORTED, "%s: heads of 16, 32, .. 256 channels", what);
    if (block_log2(block) < 0) return fail(CG_ERR_UNSUPPORTED, "%s: blocks of 16, 32, 64 or 128 positions", what);
    if (capacity < block || capacity % block || capacity > 0x7FFFFF00u) return fail(CG_ERR_SHAPE, "%s: a cache holds whole blocks, fewer than 2^31 positions", what);
    if (kv_heads < 1 || kv_heads > 4096) return fail(CG_ERR_ARG, "%s: bad head counts", what);
    const uint64_t touched = std::min(capacity / block, tokens / block + 2);
    if ((uint64_t)sequences * kv_heads * 2 * touched >= 1u << 24) return fail(CG_ERR_UNSUPPORTED, "%s: too many blocks in one call", what);
    return CG_OK;
}
int check_heads(size_t heads, size_t kv_heads, size_t tokens, float scale, const char *what) {
    if (heads < 1 || heads % kv_heads || heads > 4096) return fail(CG_ERR_ARG, "%s: bad head counts", what);
    if (heads / kv_heads * tokens >= 1u << 24) return fail(CG_ERR_UNSUPPORTED, "%s: too many rows in one call", what);
    if (!std::isfinite(scale)) return fail(CG_ERR_ARG, "%s: the scale is not a finite number", what);
    return CG_OK;
}

// A launch's threads are fewer than 2^32 (an append's workgroups have up to 512).
int check_launch(const CacheAppendPlan &p) {
    const AppendShape s = shape_cache_append(p);
    return s.groups * s.threads >= 1ull << 32 ? fail(CG_ERR_UNSUPPORTED, "cache append: too many blocks in one call") : CG_OK;
}

template <class F> int guarded(F &&f) { // (nothing is thrown through the C ABI)
    try {
        return f();
    } catch (const std::exception &e) {
        return fail(CG_ERR_DEVICE, "%s", e.what());
    }
}

// ---- tensors of a backend ----------------------------------------------------------------------------------------------

// f32 rows as the kernels take them; their pitch may be 0 (one row for all).
int activations(cg_backend *b, Held &h, cg_tensor *t, int64_t rows, int64_t features, const void **p, int64_t *pitch, const char *what) {
    Rows r;
    if (int rc = rows_of(b, h, t, rows, features, &r, what)) return rc;
    *p = r.p;
    *pitch = r.pitch;
    return CG_OK;
}

// A cache's tensor as dense memory in its format: as it lies, or a copy.
bool lies_as(const cg_tensor *t, int fmt) { return !t->uniform && !t->pend && t->buf && t->buf->fmt == fmt && is_contiguous(t) && t->split < 0; }
int copy_as(cg_backend *b, Held &h, cg_tensor *t, int fmt, cg_tensor **out) {
    if (t->split >= 0 || t->pend) {
        cg_tensor *m = nullptr;
        if (int rc = materialize(b, t, &m)) return rc;
        t = h.add(m);
    }
    cg_tensor *o = nullptr;
    if (int rc = new_dense(b, t->dt, t->dims, t->rank, &o, 0, fmt)) return rc;
    const cg_tensor *ins[1] = {t};
    if (int rc = launch_elementwise(b, kCopy, t->dt, o, ins, 1)) {
        release(o);
        return rc;
    }
    *out = o;
    return CG_OK;
}
int memory_of(const cg_tensor *t, void **p) {
    const void *at;
    int fmt;
    if (int rc = device_ptr_fmt(t, &at, &fmt)) return rc;
    *p = const_cast<void *>(at);
    return CG_OK;
}
int cache_to_read(cg_backend *b, Held &h, cg_tensor *t, int fmt, void **p) {
    if (int rc = ensure_concrete(t)) return rc;
    if (lies_as(t, fmt)) {
        if (int rc = memory_of(t, p)) return rc;
        if (at16(*p)) return CG_OK;
    }
    cg_tensor *o = nullptr;
    if (int rc = copy_as(b, h, t, fmt, &o)) return rc;
    return memory_of(h.add(o), p);
}
// The same to be written: in place where this call holds the only reference.
int cache_to_write(cg_backend *b, Held &h, cg_tensor *t, int fmt, void **p, cg_tensor **out) {
    if (int rc = ensure_concrete(t)) return rc;
    if (t->rc.load() == 1 && lies_as(t, fmt) && t->buf->rc.load() == 1 && !t->buf->rs && !t->buf->constant) {
        if (int rc = memory_of(t, p)) return rc;
        if (at16(*p)) {
            drop_packed(t->buf); // what was made of its contents
            buffer_release(t->buf->wide);
            t->buf->wide = nullptr;
            retain(t);
            *out = t;
            return CG_OK;
        }
    }
    cg_tensor *o = nullptr;
    if (int rc = copy_as(b, h, t, fmt, &o)) return rc;
    *out = o;
    return memory_of(o, p);
}

// The sizes of a cache from its tensors' shapes.
int cache_of(int64_t B, const cg_tensor *kc, const cg_tensor *vc, const cg_tensor *ks, const cg_tensor *vs, Cache8 *c, const char *what) {
    if (kc->dt != CG_F8 || vc->dt != CG_F8 || ks->dt != CG_F32 || vs->dt != CG_F32) return fail(CG_ERR_DTYPE, "%s: codes are f8, scales f32", what);
    if (kc->rank != 4 || vc->rank != 5 || ks->rank != 3 || vs->rank != 3) return fail(CG_ERR_SHAPE, "%s: bad ranks", what);
    const int64_t G = kc->dims[1], C = kc->dims[2], D = kc->dims[3], nb = vc->dims[2], V = vc->dims[3], n = vc->dims[4];
    if (kc->dims[0] != B || vc->dims[0] != B || vc->dims[1] != G || nb < 1 || n < 1 || nb * n != C) return fail(CG_ERR_SHAPE, "%s: incompatible caches", what);
    for (const cg_tensor *s : {ks, vs})
        if (s->dims[0] != B || s->dims[1] != G || s->dims[2] != nb) return fail(CG_ERR_SHAPE, "%s: incompatible scales", what);
    *c = {};
    c->kv_heads = (uint32_t)G;
    c->dim = (uint32_t)D;
    c->vdim = (uint32_t)V;
    c->capacity = (uint32_t)C;
    c->block_log2 = (uint32_t)block_log2((size_t)n);
    return G < 0 || C > 0x7FFFFF00 ? fail(CG_ERR_UNSUPPORTED, "%s: too long a cache", what) : CG_OK;
}

TokenBatch batch_of(int64_t B, int64_t S, uint64_t position) { return {(uint32_t)B, (uint32_t)S, position, nullptr, nullptr}; }

// The frequencies of a rotation in memory, kept by the backend.
int turns_of(cg_backend *b, const cg_rotation &r, const double **turns, float *magnitude) {
    cg_rotation key; // (every byte of it: they are compared)
    memset(&key, 0, sizeof key);
    key.dims = r.dims;
    key.interleaved = r.interleaved != 0;
    key.scaling = r.scaling;
    key.base = r.base;
    key.factor = r.factor;
    key.low = r.low;
    key.high = r.high;
    key.original = r.original;
    key.magnitude = r.magnitude;
    for (const TurnTable &t : b->turn_tables)
        if (memcmp(&t.of, &key, sizeof key) == 0) {
            *turns = static_cast<const double *>(t.turns->ptr);
            *magnitude = t.magnitude;
            return CG_OK;
        }
    double host[256];
    TurnTable t;
    if (int rc = cg_rotation_turns(&r, host, &t.magnitude)) return rc;
    memcpy(&t.of, &key, sizeof key);
    b->turn_tables.reserve(kMostTurnTables);
    Buffer *buf = new Buffer;
    buf->be = b;
    buf->elems = (int64_t)r.dims; // words
    int rc = b->pool.alloc(r.dims * 4, &buf->ptr, &buf->cls);
    if (!rc) rc = launch_rotation_table(LaunchOn{&b->stream, nullptr}, host, (uint32_t)(r.dims / 2), static_cast<double *>(buf->ptr));
    if (rc) {
        buffer_release(buf);
        return rc;
    }
    if (b->turn_tables.size() == kMostTurnTables) { // (stream-ordered)
        buffer_release(b->turn_tables.front().turns);
        b->turn_tables.erase(b->turn_tables.begin());
    }
    t.turns = buf;
    b->turn_tables.push_back(t);
    *turns = static_cast<const double *>(buf->ptr);
    *magnitude = t.magnitude;
    return CG_OK;
}

// ---- a caller's memory -------------------------------------------------------------------------------------------------

std::atomic<bool> g_loaded[64] = {};

// The calling thread's device for the duration of a call.
struct OnDevice {
    int prev = -1, device;
    explicit OnDevice(int d) : device(d) {}
    int enter() {
        if (device < 0 || device >= 64 || !g_loaded[device].load(std::memory_order_acquire))
            return fail(CG_ERR_ARG, "device %d is not set up (call cg_noalloc_setup or cg_backend_create on it first, outside any stream capture)", device);
        CG_HIP(hipGetDevice(&prev));
        if (prev != device) CG_HIP(hipSetDevice(device));
        return CG_OK;
    }
    ~OnDevice() {
        if (prev >= 0 && prev != device) (void)hipSetDevice(prev);
    }
};

size_t element_bytes(cg_dtype dt) { return dt == CG_F32 ? 4 : dt == CG_F16 || dt == CG_BF16 ? 2 : 0; }
int check_elements(cg_dtype dt, std::initializer_list<const void *> arrays, const char *what) {
    const size_t n = element_bytes(dt);
    if (!n) return fail(CG_ERR_DTYPE, "%s: elements are f32, f16 or bf16", what);
    for (const void *p : arrays)
        if (reinterpret_cast<uintptr_t>(p) % n) return fail(CG_ERR_ARG, "%s: an array is not at a multiple of its elements' size", what);
    return CG_OK;
}
int pitch_of(size_t pitch, size_t width, int64_t *out, const char *what) {
    if (pitch && (pitch < width || pitch > 1u << 30)) return fail(CG_ERR_ARG, "%s: rows lie closer than they are wide, or too far apart", what);
    *out = (int64_t)(pitch ? pitch : width);
    return CG_OK;
}
bool no_tokens(const cg_token_batch &a) { return a.sequences == 0 || a.tokens == 0; }
int batch_from(const cg_token_batch &a, TokenBatch *b, const char *what) {
    if (int rc = check_batch(a.sequences, a.tokens, a.held ? 0 : a.position, what)) return rc;
    if (reinterpret_cast<uintptr_t>(a.held) % 4 || reinterpret_cast<uintptr_t>(a.counts) % 4) return fail(CG_ERR_ARG, "%s: lengths are u32 at multiples of 4 bytes", what);
    *b = {(uint32_t)a.sequences, (uint32_t)a.tokens, a.position, a.held, a.counts};
    return CG_OK;
}
int cache_from(const cg_cache8 &a, size_t sequences, size_t tokens, Cache8 *c, bool memory, const char *what) {
    if (int rc = check_cache(sequences, tokens, a.kv_heads, a.dim, a.vdim, a.capacity, a.block, what)) return rc;
    if (memory) {
        if (!a.k_codes || !a.v_codes || !a.k_scale || !a.v_scale) return fail(CG_ERR_ARG, "%s: null argument", what);
        if (!at16(a.k_codes) || !at16(a.v_codes)) return fail(CG_ERR_ARG, "%s: codes lie at multiples of 16 bytes", what);
        if (reinterpret_cast<uintptr_t>(a.k_scale) % 4 || reinterpret_cast<uintptr_t>(a.v_scale) % 4) return fail(CG_ERR_ARG, "%s: scales lie at multiples of 4 bytes", what);
    }
    *c = {a.k_codes, a.v_codes, a.k_scale, a.v_scale, (uint32_t)a.kv_heads, (uint32_t)a.dim, (uint32_t)a.vdim, (uint32_t)a.capacity, (uint32_t)block_log2(a.block)};
    return CG_OK;
}
int attention_from(const cg_cache_attention_rows &a, bool memory, CacheAttentionPlan *p) {
    const char *const what = "cache attention";
    *p = {};
    if (int rc = check_elements(a.dtype, {a.q, a.out}, what)) return rc;
    if (int rc = batch_from(a.batch, &p->batch, what)) return rc;
    if (int rc = cache_from(a.cache, a.batch.sequences, a.batch.tokens, &p->cache, memory, what)) return rc;
    if (int rc = check_heads(a.heads, a.cache.kv_heads, a.batch.tokens, a.scale, what)) return rc;
    if (int rc = pitch_of(a.q_pitch, a.heads * a.cache.dim, &p->q_pitch, what)) return rc;
    if (int rc = pitch_of(a.out_pitch, a.heads * a.cache.vdim, &p->out_pitch, what)) return rc;
    p->q = a.q;
    p->out = a.out;
    p->heads = (uint32_t)a.heads;
    p->rep = (uint32_t)(a.heads / a.cache.kv_heads);
    p->window = a.window;
    p->scale = a.scale;
    return CG_OK;
}
// The workgroups of a shaped plan's launches.
int check_launch(const CacheAttentionPlan &p) {
    if ((uint64_t)p.bgs * p.row_blocks * p.splits >= 1u << 24 || (uint64_t)p.bgs * p.rows >= 1u << 28) return fail(CG_ERR_UNSUPPORTED, "cache attention: too many rows in one call");
    return CG_OK;
}

} // namespace

int cache_noalloc_setup(int device) {
    if (int rc = load_rotary_kernels()) return rc;
    if (int rc = load_cache_append_kernels()) return rc;
    if (int rc = load_cache_attention_kernels()) return rc;
    g_loaded[device].store(true, std::memory_order_release);
    return CG_OK;
}

} // namespace cg

using namespace cg;

extern "C" {

int cg_rotation_turns(const cg_rotation *r, double *turns, float *magnitude) {
    if (!r || !turns || !magnitude) return fail(CG_ERR_ARG, "null argument");
    const double pi2 = 6.283185307179586476925286766559;
    const size_t half = r->dims / 2;
    if (r->dims < 2 || r->dims % 2 || r->dims > 512) return fail(CG_ERR_ARG, "rotation: an even number of values up to 512 of a head is turned");
    if (!(r->base > 0.0) || !std::isfinite(r->base) || !(r->magnitude >= 0.0) || !std::isfinite(r->magnitude)) return fail(CG_ERR_ARG, "rotation: bad base or magnitude");
    const bool linear = r->scaling == CG_ROTATION_LINEAR, bands = r->scaling == CG_ROTATION_BANDS, ramp = r->scaling == CG_ROTATION_RAMP;
    if (!linear && !bands && !ramp && r->scaling != CG_ROTATION_PLAIN) return fail(CG_ERR_ARG, "rotation: unknown scaling");
    if ((linear || bands || ramp) && (!(r->factor > 0.0) || !std::isfinite(r->factor))) return fail(CG_ERR_ARG, "rotation: bad factor");
    if ((bands || ramp) && (!(r->original > 0.0) || !std::isfinite(r->original) || !(r->low > 0.0) || !(r->high > r->low) || !std::isfinite(r->high)))
        return fail(CG_ERR_ARG, "rotation: bad limits");
    if (ramp && r->base <= 1.0) return fail(CG_ERR_ARG, "rotation: bad base");
    double from = 0.0, to = 1.0;
    if (ramp) {
        auto pair_of = [&](double times) { return (double)r->dims * std::log(r->original / (times * pi2)) / (2.0 * std::log(r->base)); };
        from = std::max(std::floor(pair_of(r->high)), 0.0);
        to = std::max(std::min(std::ceil(pair_of(r->low)), (double)r->dims - 1.0), from + 1e-3);
    }
    for (size_t i = 0; i < half; i++) {
        double f = std::pow(r->base, -2.0 * (double)i / (double)r->dims), part = 0.0; // part: of f that stays
        if (linear) part = 0.0;
        else if (bands) part = (r->original * f / pi2 - r->low) / (r->high - r->low);
        else if (ramp) part = 1.0 - ((double)i - from) / (to - from);
        else part = 1.0;
        part = std::min(std::max(part, 0.0), 1.0);
        if (part < 1.0) f *= part + (1.0 - part) / r->factor;
        turns[i] = f / pi2;
    }
    *magnitude = (float)(r->magnitude > 0.0 ? r->magnitude : ramp ? 0.1 * std::log(r->factor) + 1.0 : 1.0);
    return CG_OK;
}

int cg_block_rotary(cg_backend *b, const cg_rotary_args *a, cg_tensor **q_out, cg_tensor **k_out) {
    Enter entered(b);
    if (!a) return fail(CG_ERR_ARG, "null argument");
    return guarded([&]() -> int {
        Held h;
        for (cg_tensor *t : {a->q, a->k}) h.add(t);
        if (!a->q || !q_out || (a->k && !k_out)) return fail(CG_ERR_ARG, "null argument");
        CG_ENTER_BLOCK(b);
        const char *const what = "block_rotary";
        if (int rc = check_rotation(a->heads, a->k ? a->kv_heads : 0, a->dim, a->rotation.dims, what)) return rc;
        if (a->k && a->kv_heads < 1) return fail(CG_ERR_ARG, "%s: bad head counts or sizes", what);
        if (a->q->rank != 3 || (a->k && a->k->rank != 3)) return fail(CG_ERR_SHAPE, "%s: bad ranks", what);
        const int64_t B = a->q->dims[0], S = a->q->dims[1];
        if (B < 1 || S < 1) return fail(CG_ERR_SHAPE, "%s: no tokens", what);
        if (int rc = check_batch((size_t)B, (size_t)S, a->position, what)) return rc;
        RotaryPlan p{};
        p.batch = batch_of(B, S, a->position);
        p.heads = (uint32_t)a->heads;
        p.kv_heads = (uint32_t)(a->k ? a->kv_heads : 0);
        p.dim = (uint32_t)a->dim;
        p.rot = (uint32_t)a->rotation.dims;
        p.interleaved = a->rotation.interleaved != 0;
        p.q_out_pitch = (int64_t)(a->heads * a->dim);
        p.k_out_pitch = (int64_t)(p.kv_heads * a->dim);
        if (a->k && (a->k->dims[0] != B || a->k->dims[1] != S)) return fail(CG_ERR_SHAPE, "%s: q and k have different tokens", what);
        if (int rc = activations(b, h, a->q, B * S, p.q_out_pitch, &p.q, &p.q_pitch, what)) return rc;
        if (a->k)
            if (int rc = activations(b, h, a->k, B * S, p.k_out_pitch, &p.k, &p.k_pitch, what)) return rc;
        if (int rc = turns_of(b, a->rotation, &p.turns, &p.magnitude)) return rc;
        const int64_t qd[3] = {B, S, p.q_out_pitch}, kd[3] = {B, S, p.k_out_pitch};
        cg_tensor *qo = nullptr, *ko = nullptr;
        int rc = new_dense(b, CG_F32, qd, 3, &qo);
        if (!rc && a->k) rc = new_dense(b, CG_F32, kd, 3, &ko);
        if (!rc) {
            p.q_out = qo->buf->ptr;
            if (ko) p.k_out = ko->buf->ptr;
            rc = launch_rotary(LaunchOn{&b->stream, nullptr}, CG_F32, p);
        }
        if (rc) {
            release(qo);
            release(ko);
            return rc;
        }
        *q_out = qo;
        if (a->k) *k_out = ko;
        return CG_OK;
    });
}

int cg_block_cache_append(cg_backend *b, const cg_cache_append_args *a, cg_tensor **k_codes_out, cg_tensor **v_codes_out, cg_tensor **k_scale_out,
                          cg_tensor **v_scale_out) {
    Enter entered(b);
    if (!a) return fail(CG_ERR_ARG, "null argument");
    return guarded([&]() -> int {
        Held h;
        for (cg_tensor *t : {a->k, a->v, a->k_codes, a->v_codes, a->k_scale, a->v_scale}) h.add(t);
        if (!a->k || !a->v || !a->k_codes || !a->v_codes || !a->k_scale || !a->v_scale || !k_codes_out || !v_codes_out || !k_scale_out || !v_scale_out)
            return fail(CG_ERR_ARG, "null argument");
        CG_ENTER_BLOCK(b);
        const char *const what = "block_cache_append";
        if (a->k->rank != 3 || a->v->rank != 3) return fail(CG_ERR_SHAPE, "%s: bad ranks", what);
        const int64_t B = a->k->dims[0], S = a->k->dims[1];
        if (B < 1 || S < 1) return fail(CG_ERR_SHAPE, "%s: no tokens", what);
        if (int rc = check_batch((size_t)B, (size_t)S, a->position, what)) return rc;
        CacheAppendPlan p{};
        if (int rc = cache_of(B, a->k_codes, a->v_codes, a->k_scale, a->v_scale, &p.cache, what)) return rc;
        const Cache8 &c = p.cache;
        if (int rc = check_cache((size_t)B, (size_t)S, c.kv_heads, c.dim, c.vdim, c.capacity, (size_t)a->v_codes->dims[4], what)) return rc;
        if (a->position + (uint64_t)S > c.capacity) return fail(CG_ERR_RANGE, "%s: the cache has no room for the positions", what);
        if (a->v->dims[0] != B || a->v->dims[1] != S) return fail(CG_ERR_SHAPE, "%s: k and v have different tokens", what);
        p.batch = batch_of(B, S, a->position);
        if (int rc = check_launch(p)) return rc;
        if (int rc = activations(b, h, a->k, B * S, (int64_t)c.kv_heads * c.dim, &p.k, &p.k_pitch, what)) return rc;
        if (int rc = activations(b, h, a->v, B * S, (int64_t)c.kv_heads * c.vdim, &p.v, &p.v_pitch, what)) return rc;
        cg_tensor *o[4] = {};
        void *m[4] = {};
        cg_tensor *const in[4] = {a->k_codes, a->v_codes, a->k_scale, a->v_scale};
        int rc = CG_OK;
        for (int i = 0; i < 4 && !rc; i++) rc = cache_to_write(b, h, in[i], i < 2 ? kFmtF8 : kFmtWords, &m[i], &o[i]);
        if (!rc) {
            p.cache.k_codes = static_cast<uint8_t *>(m[0]);
            p.cache.v_codes = static_cast<uint8_t *>(m[1]);
            p.cache.k_scale = static_cast<float *>(m[2]);
            p.cache.v_scale = static_cast<float *>(m[3]);
            rc = launch_cache_append(LaunchOn{&b->stream, nullptr}, CG_F32, p);
        }
        if (rc) {
            for (cg_tensor *t : o) release(t);
            return rc;
        }
        *k_codes_out = o[0];
        *v_codes_out = o[1];
        *k_scale_out = o[2];
        *v_scale_out = o[3];
        return CG_OK;
    });
}

int cg_block_cache_attention(cg_backend *b, const cg_cache_attention_args *a, cg_tensor **out) {
    Enter entered(b);
    if (!a) return fail(CG_ERR_ARG, "null argument");
    return guarded([&]() -> int {
        Held h;
        for (cg_tensor *t : {a->q, a->k_codes, a->v_codes, a->k_scale, a->v_scale}) h.add(t);
        if (!a->q || !a->k_codes || !a->v_codes || !a->k_scale || !a->v_scale || !out) return fail(CG_ERR_ARG, "null argument");
        CG_ENTER_BLOCK(b);
        const char *const what = "block_cache_attention";
        if (a->q->rank != 3) return fail(CG_ERR_SHAPE, "%s: bad ranks", what);
        const int64_t B = a->q->dims[0], S = a->q->dims[1];
        if (B < 1 || S < 1) return fail(CG_ERR_SHAPE, "%s: no tokens", what);
        if (int rc = check_batch((size_t)B, (size_t)S, a->position, what)) return rc;
        CacheAttentionPlan p{};
        if (int rc = cache_of(B, a->k_codes, a->v_codes, a->k_scale, a->v_scale, &p.cache, what)) return rc;
        const Cache8 &c = p.cache;
        if (int rc = check_cache((size_t)B, (size_t)S, c.kv_heads, c.dim, c.vdim, c.capacity, (size_t)a->v_codes->dims[4], what)) return rc;
        if (int rc = check_heads(a->heads, c.kv_heads, (size_t)S, a->scale, what)) return rc;
        if (a->position + (uint64_t)S > c.capacity) return fail(CG_ERR_RANGE, "%s: the cache does not hold the positions", what);
        p.batch = batch_of(B, S, a->position);
        p.heads = (uint32_t)a->heads;
        p.rep = p.heads / c.kv_heads;
        p.window = a->window;
        p.scale = a->scale;
        p.out_pitch = (int64_t)p.heads * c.vdim;
        if (int rc = activations(b, h, a->q, B * S, (int64_t)p.heads * c.dim, &p.q, &p.q_pitch, what)) return rc;
        void *m[4] = {};
        cg_tensor *const in[4] = {a->k_codes, a->v_codes, a->k_scale, a->v_scale};
        for (int i = 0; i < 4; i++)
            if (int rc = cache_to_read(b, h, in[i], i < 2 ? kFmtF8 : kFmtWords, &m[i])) return rc;
        p.cache.k_codes = static_cast<uint8_t *>(m[0]);
        p.cache.v_codes = static_cast<uint8_t *>(m[1]);
        p.cache.k_scale = static_cast<float *>(m[2]);
        p.cache.v_scale = static_cast<float *>(m[3]);
        const size_t bytes = shape_cache_attention(&p);
        if (int rc = check_launch(p)) return rc;
        Scratch tmp(b);
        if (bytes) {
            void *w = nullptr;
            if (int rc = tmp.get(bytes, &w)) return rc;
            p.parts = static_cast<float *>(w);
            p.stats = reinterpret_cast<float2 *>(p.parts + (size_t)p.bgs * p.splits * p.rows * c.vdim);
        }
        const int64_t od[3] = {B, S, p.out_pitch};
        cg_tensor *o = nullptr;
        int rc = new_dense(b, CG_F32, od, 3, &o);
        if (!rc) {
            p.out = o->buf->ptr;
            rc = launch_cache_attention(LaunchOn{&b->stream, nullptr}, CG_F32, p);
        }
        if (rc) {
            release(o);
            return rc;
        }
        *out = o;
        return CG_OK;
    });
}

int cg_rotary_noalloc(int device, const cg_rotary_rows *a, void *stream) {
    const char *const what = "rotary";
    if (!a) return fail(CG_ERR_ARG, "null argument");
    RotaryPlan p{};
    if (int rc = check_elements(a->dtype, {a->q, a->k, a->q_out, a->k_out}, what)) return rc;
    if (int rc = batch_from(a->batch, &p.batch, what)) return rc;
    if (int rc = check_rotation(a->heads, a->k ? a->kv_heads : 0, a->dim, a->rot_dims, what)) return rc;
    if (a->k && a->kv_heads < 1) return fail(CG_ERR_ARG, "%s: bad head counts or sizes", what);
    if (no_tokens(a->batch)) return CG_OK;
    if (!a->q || !a->q_out || (a->k && !a->k_out) || !a->turns) return fail(CG_ERR_ARG, "%s: null argument", what);
    if (reinterpret_cast<uintptr_t>(a->turns) % 8) return fail(CG_ERR_ARG, "%s: turns lie at multiples of 8 bytes", what);
    const size_t qw = a->heads * a->dim, kw = (a->k ? a->kv_heads : 0) * a->dim;
    if (int rc = pitch_of(a->q_pitch, qw, &p.q_pitch, what)) return rc;
    if (int rc = pitch_of(a->q_out_pitch, qw, &p.q_out_pitch, what)) return rc;
    if (int rc = pitch_of(a->k ? a->k_pitch : 0, kw, &p.k_pitch, what)) return rc;
    if (int rc = pitch_of(a->k ? a->k_out_pitch : 0, kw, &p.k_out_pitch, what)) return rc;
    if ((a->q == a->q_out && p.q_pitch != p.q_out_pitch) || (a->k && a->k == a->k_out && p.k_pitch != p.k_out_pitch))
        return fail(CG_ERR_ARG, "%s: results in place of their operand have its pitch", what);
    p.q = a->q;
    p.k = a->k;
    p.q_out = a->q_out;
    p.k_out = a->k ? a->k_out : nullptr;
    p.heads = (uint32_t)a->heads;
    p.kv_heads = (uint32_t)(a->k ? a->kv_heads : 0);
    p.dim = (uint32_t)a->dim;
    p.rot = (uint32_t)a->rot_dims;
    p.interleaved = a->interleaved != 0;
    p.magnitude = a->magnitude;
    p.turns = a->turns;
    OnDevice on(device);
    if (int rc = on.enter()) return rc;
    return launch_rotary(LaunchOn{nullptr, static_cast<hipStream_t>(stream)}, a->dtype, p);
}

int cg_cache_append_noalloc(int device, const cg_cache_append_rows *a, void *stream) {
    const char *const what = "cache append";
    if (!a) return fail(CG_ERR_ARG, "null argument");
    CacheAppendPlan p{};
    if (int rc = check_elements(a->dtype, {a->k, a->v}, what)) return rc;
    if (int rc = batch_from(a->batch, &p.batch, what)) return rc;
    if (no_tokens(a->batch)) return CG_OK;
    if (int rc = cache_from(a->cache, a->batch.sequences, a->batch.tokens, &p.cache, true, what)) return rc;
    if (!a->k || !a->v) return fail(CG_ERR_ARG, "%s: null argument", what);
    if (int rc = pitch_of(a->k_pitch, a->cache.kv_heads * a->cache.dim, &p.k_pitch, what)) return rc;
    if (int rc = pitch_of(a->v_pitch, a->cache.kv_heads * a->cache.vdim, &p.v_pitch, what)) return rc;
    if (int rc = check_launch(p)) return rc;
    p.k = a->k;
    p.v = a->v;
    OnDevice on(device);
    if (int rc = on.enter()) return rc;
    return launch_cache_append(LaunchOn{nullptr, static_cast<hipStream_t>(stream)}, a->dtype, p);
}

int cg_cache_attention_workspace(const cg_cache_attention_rows *a, size_t *bytes) {
    if (!a || !bytes) return fail(CG_ERR_ARG, "null argument");
    *bytes = 0;
    if (no_tokens(a->batch)) return CG_OK;
    CacheAttentionPlan p;
    if (int rc = attention_from(*a, false, &p)) return rc;
    const size_t n = shape_cache_attention(&p);
    if (int rc = check_launch(p)) return rc;
    *bytes = n;
    return CG_OK;
}

int cg_cache_attention_noalloc(int device, const cg_cache_attention_rows *a, void *stream) {
    const char *const what = "cache attention";
    if (!a) return fail(CG_ERR_ARG, "null argument");
    if (no_tokens(a->batch)) return CG_OK;
    CacheAttentionPlan p;
    if (int rc = attention_from(*a, true, &p)) return rc;
    if (!a->q || !a->out) return fail(CG_ERR_ARG, "%s: null argument", what);
    const size_t bytes = shape_cache_attention(&p);
    if (int rc = check_launch(p)) return rc;
    if (bytes && (!a->workspace || a->workspace_bytes < bytes)) return fail(CG_ERR_ARG, "%s: needs a workspace of %zu bytes", what, bytes);
    if (bytes && !at16(a->workspace)) return fail(CG_ERR_ARG, "%s: the workspace lies at a multiple of 16 bytes", what);
    if (bytes) {
        p.parts = static_cast<float *>(a->workspace);
        p.stats = reinterpret_cast<float2 *>(p.parts + (size_t)p.bgs * p.splits * p.rows * p.cache.vdim);
    }
    OnDevice on(device);
    if (int rc = on.enter()) return rc;
    return launch_cache_attention(LaunchOn{nullptr, static_cast<hipStream_t>(stream)}, a->dtype, p);
}

} // extern "C"
