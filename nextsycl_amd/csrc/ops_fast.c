/* ops_fast.c: the size checks and the call of attn.Ops.decode / prompt / pre_store, and of a token's calls of a layer beside
 * attention (ssm_step, norm_gated, norm_residual, q4_product) and over an 8-bit cache in blocks (kv8_store, kv8_attend), in one step of native code.
 *
 * A short context's step is a few microseconds of GPU work, and the wrappers' checks and ctypes' conversion of 18 - 28 arguments
 * took longer than a launch: a token's two calls 15.2 us, of them 10 for three launches. Each function here takes the addresses
 * of the library's entry points, the GPU's handle and the wrapper's own arguments. It returns False and has called nothing
 * where a check fails or an argument is not the plain kind (int, float, a buffer of int ptr and len): the wrapper then goes the
 * general way, which says what is wrong. Else it makes the call, once, and returns True or, where that failed, the library's number:
 * a call may fail behind launches it has made, so the wrapper raises and makes no second one. */
#define Py_LIMITED_API 0x030A0000
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "ns_attn.h"
#include "ns_kv8.h"
#include "ns_layer.h"
#include "ns_pre.h"

static PyObject *s_ptr, *s_len;

typedef struct {
    void *ptr;
    int64_t len;
} buf_t;

/* what a function returns for a call it has made */
static PyObject *made(int rc) {
    if (rc == 0) Py_RETURN_TRUE;
    return PyLong_FromLong(rc);
}

/* sizes up to 2^31: the products below then fit 128 bits */
static int get_size(PyObject *o, int64_t *v) {
    if (!PyLong_Check(o)) return 0;
    *v = PyLong_AsLongLong(o);
    if (*v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return 0;
    }
    return *v >= 0 && *v <= (int64_t) 1 << 31;
}
static int get_float(PyObject *o, float *v) {
    if (!PyFloat_Check(o) && !PyLong_Check(o)) return 0;
    const double d = PyFloat_AsDouble(o);
    if (d == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return 0;
    }
    *v = (float) d;
    return 1;
}
static int get_address(PyObject *o, void **v) {
    if (!PyLong_Check(o)) return 0;
    *v = PyLong_AsVoidPtr(o);
    if (!*v) PyErr_Clear();
    return *v != NULL;
}
static int get_buf(PyObject *o, buf_t *b) {
    PyObject *p = PyObject_GetAttr(o, s_ptr), *n = p ? PyObject_GetAttr(o, s_len) : NULL;
    int ok = 0;
    if (p && n && get_address(p, &b->ptr) && PyLong_Check(n)) {
        b->len = PyLong_AsLongLong(n);
        ok = !(b->len == -1 && PyErr_Occurred());
    }
    Py_XDECREF(p);
    Py_XDECREF(n);
    if (!ok) PyErr_Clear();
    return ok;
}

static int64_t elt(int64_t qt) { return qt == 0 ? 4 : qt <= 2 ? 2 : -1; }
static int64_t row_bytes(int64_t kt, int64_t D) { return kt == 1 ? D + D / 32 * 2 : kt == 2 ? D / 2 + D / 32 * 2 : kt == 0 || kt == 3 ? 2 * D : -1; }
/* whether b holds (rows - 1) stride + last elements of e bytes, or n elements */
static int holds(const buf_t *b, int64_t rows, int64_t stride, int64_t last, int64_t e) {
    return (__int128) b->len >= ((__int128) (rows - 1) * stride + last) * e;
}
static int holds3(const buf_t *b, int64_t x, int64_t y, int64_t z) { return (__int128) b->len >= (__int128) x * y * z; }

/* what decode and prompt share: (.., handle, qt, kt, q, qs, kc, vc, T, Hq, Hkv, D, cap, p0, out, ..) */
typedef struct {
    void *g;
    int64_t qt, kt, qs, T, Hq, Hkv, D, cap, p0;
    buf_t q, kc, vc, out;
} pass_t;
static int get_pass(PyObject *const *a, pass_t *p) {
    if (!get_address(a[0], &p->g) || !get_size(a[1], &p->qt) || !get_size(a[2], &p->kt) || !get_buf(a[3], &p->q) || !get_size(a[4], &p->qs) ||
        !get_buf(a[5], &p->kc) || !get_buf(a[6], &p->vc) || !get_size(a[7], &p->T) || !get_size(a[8], &p->Hq) || !get_size(a[9], &p->Hkv) ||
        !get_size(a[10], &p->D) || !get_size(a[11], &p->cap) || !get_size(a[12], &p->p0) || !get_buf(a[13], &p->out))
        return 0;
    const int64_t e = elt(p->qt), rb = row_bytes(p->kt, p->D);
    return e > 0 && rb >= 0 && p->T > 0 && holds(&p->q, p->T, p->qs, p->Hq * p->D, e) && holds3(&p->out, p->T * e, p->Hq, p->D) &&
           holds3(&p->kc, p->Hkv, p->cap, rb) && holds3(&p->vc, p->Hkv, p->cap, rb);
}

/* decode(scratch entry, entry, handle, qt, kt, q, qs, kc, vc, T, Hq, Hkv, D, cap, p0, out, scratch, win, pm, scale) */
static PyObject *fast_decode(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    void *fs, *fd;
    pass_t p;
    buf_t sc;
    int64_t win;
    float scale;
    if (n == 20 && get_address(a[0], &fs) && get_address(a[1], &fd) && get_pass(a + 2, &p) && get_buf(a[16], &sc) && get_size(a[17], &win) &&
        PyBool_Check(a[18]) && get_float(a[19], &scale)) {
        __typeof__(&ns_attn_decode_scratch) scratch = (__typeof__(&ns_attn_decode_scratch)) fs;
        __typeof__(&ns_attn_decode_t) decode = (__typeof__(&ns_attn_decode_t)) fd;
        int rc = 0, fits;
        Py_BEGIN_ALLOW_THREADS
        fits = (__int128) sc.len >= (__int128) scratch(p.T, p.Hq, p.Hkv, p.D, p.p0, win) * 4;
        if (fits)
            rc = decode((ns_gpu *) p.g, (int) p.qt, (int) p.kt, a[18] == Py_True, p.q.ptr, p.qs, p.kc.ptr, p.vc.ptr, p.T, p.Hq, p.Hkv, p.D, p.cap, p.p0, win,
                        scale, p.out.ptr, (float *) sc.ptr);
        Py_END_ALLOW_THREADS
        if (fits) return made(rc);
    }
    Py_RETURN_FALSE;
}

/* prompt(entry, handle, qt, kt, q, qs, kc, vc, T, Hq, Hkv, D, cap, p0, out, win, pm, scale) */
static PyObject *fast_prompt(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    void *f;
    pass_t p;
    int64_t win;
    float scale;
    if (n == 18 && get_address(a[0], &f) && get_pass(a + 1, &p) && get_size(a[15], &win) && PyBool_Check(a[16]) && get_float(a[17], &scale)) {
        __typeof__(&ns_attn_prompt_t) prompt = (__typeof__(&ns_attn_prompt_t)) f;
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = prompt((ns_gpu *) p.g, (int) p.qt, (int) p.kt, a[16] == Py_True, p.q.ptr, p.qs, p.kc.ptr, p.vc.ptr, p.T, p.Hq, p.Hkv, p.D, p.cap, p.p0, win, scale,
                    p.out.ptr);
        Py_END_ALLOW_THREADS
        return made(rc);
    }
    Py_RETURN_FALSE;
}

/* pre_store(entry, handle, rope, qt, kt, ring, q, qss, qhs, qo, qos, k, kss, khs, v, vss, qw, kw, eps, n_rot, theta, T, Hq, Hkv, D, cap, p0, kc, vc) */
static PyObject *fast_pre_store(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    void *f, *g;
    buf_t q, qo, k, v, qw, kw, kc, vc;
    int64_t rope, qt, kt, qss, qhs, qos, kss, khs, vss, n_rot, T, Hq, Hkv, D, cap, p0;
    float eps, theta;
    if (n == 29 && get_address(a[0], &f) && get_address(a[1], &g) && get_size(a[2], &rope) && get_size(a[3], &qt) && get_size(a[4], &kt) && PyBool_Check(a[5]) &&
        get_buf(a[6], &q) && get_size(a[7], &qss) && get_size(a[8], &qhs) && get_buf(a[9], &qo) && get_size(a[10], &qos) && get_buf(a[11], &k) &&
        get_size(a[12], &kss) && get_size(a[13], &khs) && get_buf(a[14], &v) && get_size(a[15], &vss) && get_buf(a[16], &qw) && get_buf(a[17], &kw) &&
        get_float(a[18], &eps) && get_size(a[19], &n_rot) && get_float(a[20], &theta) && get_size(a[21], &T) && get_size(a[22], &Hq) &&
        get_size(a[23], &Hkv) && get_size(a[24], &D) && get_size(a[25], &cap) && get_size(a[26], &p0) && get_buf(a[27], &kc) && get_buf(a[28], &vc)) {
        const int64_t e = elt(qt), rb = row_bytes(kt, D);
        if (e > 0 && rb >= 0 && T > 0 && Hq > 0 && Hkv > 0 && holds(&q, T, qss, (Hq - 1) * qhs + D, 4) && holds(&qo, T, qos, Hq * D, e) &&
            holds(&k, T, kss, (Hkv - 1) * khs + D, 4) && holds(&v, T, vss, Hkv * D, 4) && qw.len >= D * 4 && kw.len >= D * 4 &&
            holds3(&kc, Hkv, cap, rb) && holds3(&vc, Hkv, cap, rb)) {
            __typeof__(&ns_attn_pre_store) pre = (__typeof__(&ns_attn_pre_store)) f;
            int rc;
            Py_BEGIN_ALLOW_THREADS
            rc = pre((ns_gpu *) g, (int) rope, (int) qt, (int) kt, a[5] == Py_True, (const float *) q.ptr, qss, qhs, qo.ptr, qos, (const float *) k.ptr, kss, khs,
                     (const float *) v.ptr, vss, (const float *) qw.ptr, (const float *) kw.ptr, eps, n_rot, theta, T, Hq, Hkv, D, cap, p0, kc.ptr, vc.ptr);
            Py_END_ALLOW_THREADS
            return made(rc);
        }
    }
    Py_RETURN_FALSE;
}

/* a buffer, or None: a null pointer that any size fits */
static int get_opt(PyObject *o, buf_t *b) {
    if (o != Py_None) return get_buf(o, b);
    b->ptr = NULL;
    b->len = INT64_MAX;
    return 1;
}
static int fits(const buf_t *b, __int128 bytes) { return (__int128) b->len >= bytes; }

/* norm_gated(entry, handle, qt, y, ys, z, zs, w, out, os, T, D, groups, eps, order) */
static PyObject *fast_norm_gated(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    void *f, *g;
    buf_t y, z, w, out;
    int64_t qt, ys, zs, os, T, D, groups, order;
    float eps;
    if (n == 15 && get_address(a[0], &f) && get_address(a[1], &g) && get_size(a[2], &qt) && get_buf(a[3], &y) && get_size(a[4], &ys) && get_buf(a[5], &z) &&
        get_size(a[6], &zs) && get_opt(a[7], &w) && get_buf(a[8], &out) && get_size(a[9], &os) && get_size(a[10], &T) && get_size(a[11], &D) &&
        get_size(a[12], &groups) && get_float(a[13], &eps) && get_size(a[14], &order)) {
        const int64_t e = elt(qt);
        if (e > 0 && T > 0 && holds(&y, T, ys, D, e) && holds(&z, T, zs, D, e) && holds(&out, T, os, D, e) && fits(&w, (__int128) D * 4)) {
            __typeof__(&ns_norm_gated) call = (__typeof__(&ns_norm_gated)) f;
            int rc;
            Py_BEGIN_ALLOW_THREADS
            rc = call((ns_gpu *) g, (int) qt, y.ptr, ys, z.ptr, zs, (const float *) w.ptr, out.ptr, os, T, D, groups, eps, (int) order);
            Py_END_ALLOW_THREADS
            return made(rc);
        }
    }
    Py_RETURN_FALSE;
}

/* norm_residual(entry, handle, qt, rt, x, xs, h, hs, h1, h1s, out, os, T, D, eps, scale, post, gate, pre) */
static PyObject *fast_norm_residual(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    void *f, *g;
    buf_t x, h, h1, out, post, gate, pre;
    int64_t qt, rt, xs, hs, h1s, os, T, D;
    float eps, scale;
    if (n == 19 && get_address(a[0], &f) && get_address(a[1], &g) && get_size(a[2], &qt) && get_size(a[3], &rt) && get_opt(a[4], &x) && get_size(a[5], &xs) &&
        get_buf(a[6], &h) && get_size(a[7], &hs) && get_opt(a[8], &h1) && get_size(a[9], &h1s) && get_opt(a[10], &out) && get_size(a[11], &os) &&
        get_size(a[12], &T) && get_size(a[13], &D) && get_float(a[14], &eps) && get_float(a[15], &scale) && get_opt(a[16], &post) && get_opt(a[17], &gate) &&
        get_opt(a[18], &pre)) {
        const int64_t e = elt(qt), r = elt(rt);
        const __int128 w = (__int128) D * 4;
        if (e > 0 && r > 0 && T > 0 && (!x.ptr || holds(&x, T, xs, D, e)) && holds(&h, T, hs, D, r) && (!h1.ptr || holds(&h1, T, h1s, D, r)) &&
            (!out.ptr || holds(&out, T, os, D, e)) && fits(&post, w) && fits(&gate, w) && fits(&pre, w)) {
            __typeof__(&ns_norm_residual) call = (__typeof__(&ns_norm_residual)) f;
            int rc;
            Py_BEGIN_ALLOW_THREADS
            rc = call((ns_gpu *) g, (int) qt, (int) rt, x.ptr, xs, h.ptr, hs, h1.ptr, h1s, out.ptr, os, T, D, eps, scale, (const float *) post.ptr,
                      (const float *) gate.ptr, (const float *) pre.ptr);
            Py_END_ALLOW_THREADS
            return made(rc);
        }
    }
    Py_RETURN_FALSE;
}

/* q4_product(bytes entry, entry, handle, qt, x, xs, w, group, y, ys, T, M, K) */
static PyObject *fast_q4_product(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    void *fb, *f, *g;
    buf_t x, w, y;
    int64_t qt, xs, group, ys, T, M, K;
    if (n == 13 && get_address(a[0], &fb) && get_address(a[1], &f) && get_address(a[2], &g) && get_size(a[3], &qt) && get_buf(a[4], &x) && get_size(a[5], &xs) &&
        get_buf(a[6], &w) && get_size(a[7], &group) && get_buf(a[8], &y) && get_size(a[9], &ys) && get_size(a[10], &T) && get_size(a[11], &M) && get_size(a[12], &K)) {
        const int64_t e = elt(qt);
        __typeof__(&ns_q4_bytes) bytes = (__typeof__(&ns_q4_bytes)) fb;
        if (e > 0 && T > 0 && M > 0 && holds(&x, T, xs, K, e) && holds(&y, T, ys, M, e) && w.len >= bytes(M, K, group)) {
            __typeof__(&ns_q4_product) call = (__typeof__(&ns_q4_product)) f;
            int rc;
            Py_BEGIN_ALLOW_THREADS
            rc = call((ns_gpu *) g, (int) qt, x.ptr, xs, w.ptr, group, y.ptr, ys, T, M, K);
            Py_END_ALLOW_THREADS
            return made(rc);
        }
    }
    Py_RETURN_FALSE;
}

/* ssm_step(entry, handle, qt, xbc, xs, dt, dts, cw, cb, a, dtb, d, conv, cap, p0, R, H, P, N, G, K, h0, h1, y, ys, nslots, slots, pos, dt_lo, dt_hi) */
static PyObject *fast_ssm_step(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    void *f, *g;
    buf_t xbc, dt, cw, cb, rate, dtb, d, conv, h0, h1, y, slots, pos;
    int64_t qt, xs, dts, cap, p0, R, H, P, N, G, K, ys, nslots;
    float lo, hi;
    if (n == 30 && get_address(a[0], &f) && get_address(a[1], &g) && get_size(a[2], &qt) && get_buf(a[3], &xbc) && get_size(a[4], &xs) && get_buf(a[5], &dt) &&
        get_size(a[6], &dts) && get_buf(a[7], &cw) && get_opt(a[8], &cb) && get_buf(a[9], &rate) && get_opt(a[10], &dtb) && get_opt(a[11], &d) &&
        get_opt(a[12], &conv) && get_size(a[13], &cap) && get_size(a[14], &p0) && get_size(a[15], &R) && get_size(a[16], &H) && get_size(a[17], &P) &&
        get_size(a[18], &N) && get_size(a[19], &G) && get_size(a[20], &K) && get_opt(a[21], &h0) && get_buf(a[22], &h1) && get_buf(a[23], &y) &&
        get_size(a[24], &ys) && get_size(a[25], &nslots) && get_opt(a[26], &slots) && get_opt(a[27], &pos) && get_float(a[28], &lo) && get_float(a[29], &hi)) {
        const int64_t e = elt(qt);
        const __int128 inner = (__int128) H * P, chan = inner + 2 * (__int128) G * N, state = inner * N * 4;
        if (e > 0 && R > 0 && chan <= (int64_t) 1 << 24 && N <= 256 && K > 0 && K <= 4 && (K == 1 || conv.ptr) && holds(&xbc, R, xs, (int64_t) chan, e) &&
            holds(&dt, R, dts, H, e) && holds(&y, R, ys, (int64_t) inner, e) && fits(&cw, chan * K * 4) && fits(&rate, (__int128) H * 4) && fits(&cb, chan * 4) &&
            fits(&dtb, (__int128) H * 4) && fits(&d, (__int128) H * 4) && (K == 1 || fits(&conv, chan * 4 * cap * nslots)) && (!h0.ptr || fits(&h0, state * nslots)) &&
            fits(&h1, state * nslots) && fits(&slots, (__int128) R * 4) && fits(&pos, (__int128) R * 4)) {
            __typeof__(&ns_ssm_step) call = (__typeof__(&ns_ssm_step)) f;
            int rc;
            Py_BEGIN_ALLOW_THREADS
            rc = call((ns_gpu *) g, (int) qt, xbc.ptr, xs, dt.ptr, dts, (const float *) cw.ptr, (const float *) cb.ptr, (const float *) rate.ptr,
                      (const float *) dtb.ptr, (const float *) d.ptr, lo, hi, (float *) conv.ptr, cap, p0, (const int32_t *) pos.ptr, (const int32_t *) slots.ptr,
                      nslots, R, H, P, N, G, K, (const float *) h0.ptr, (float *) h1.ptr, y.ptr, ys);
            Py_END_ALLOW_THREADS
            return made(rc);
        }
    }
    Py_RETURN_FALSE;
}

/* a Kv8's (form, blocks, Hkv, block, D, k, v, ks, vs) */
typedef struct {
    int64_t form, blocks, Hkv, block, D;
    buf_t k, v, ks, vs;
} kv8_t;
static int get_kv8(PyObject *const *a, kv8_t *c) {
    if (!get_size(a[0], &c->form) || !get_size(a[1], &c->blocks) || !get_size(a[2], &c->Hkv) || !get_size(a[3], &c->block) || !get_size(a[4], &c->D) ||
        !get_buf(a[5], &c->k) || !get_buf(a[6], &c->v) || !get_buf(a[7], &c->ks) || !get_buf(a[8], &c->vs))
        return 0;
    if (c->Hkv > 32767 || c->block > 128 || c->D > 256) return 0;
    const __int128 rows = (__int128) c->blocks * c->Hkv;
    return fits(&c->k, rows * c->block * c->D) && fits(&c->v, rows * c->block * c->D) && fits(&c->ks, rows * 4) && fits(&c->vs, rows * 4);
}
/* the sequences: (table, tmax, S, lens, start) */
typedef struct {
    int64_t tmax, S;
    buf_t table, lens, start;
} seqs_t;
static int get_seqs(PyObject *const *a, seqs_t *q) {
    return get_buf(a[0], &q->table) && get_size(a[1], &q->tmax) && get_size(a[2], &q->S) && get_buf(a[3], &q->lens) && get_opt(a[4], &q->start) &&
           fits(&q->table, (__int128) q->S * q->tmax * 4) && fits(&q->lens, (__int128) q->S * 4) && fits(&q->start, ((__int128) q->S + 1) * 4);
}

/* kv8_store(entry, handle, 9 of the cache, 5 of the sequences, qt, k, ks, v, vs, T, most) */
static PyObject *fast_kv8_store(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    void *f, *g;
    kv8_t c;
    seqs_t q;
    buf_t k, v;
    int64_t qt, ks, vs, T, most;
    if (n == 23 && get_address(a[0], &f) && get_address(a[1], &g) && get_kv8(a + 2, &c) && get_seqs(a + 11, &q) && get_size(a[16], &qt) && get_buf(a[17], &k) &&
        get_size(a[18], &ks) && get_buf(a[19], &v) && get_size(a[20], &vs) && get_size(a[21], &T) && get_size(a[22], &most)) {
        const int64_t e = elt(qt), w = c.Hkv * c.D;
        if (e > 0 && T > 0 && holds(&k, T, ks, w, e) && holds(&v, T, vs, w, e)) {
            __typeof__(&ns_kv8_store) call = (__typeof__(&ns_kv8_store)) f;
            int rc;
            Py_BEGIN_ALLOW_THREADS
            rc = call((ns_gpu *) g, (int) c.form, (int) qt, k.ptr, ks, v.ptr, vs, T, (const int32_t *) q.start.ptr, (const int32_t *) q.lens.ptr, q.S, most,
                      (const int32_t *) q.table.ptr, q.tmax, c.Hkv, c.D, c.block, c.blocks, c.k.ptr, c.v.ptr, (float *) c.ks.ptr, (float *) c.vs.ptr);
            Py_END_ALLOW_THREADS
            return made(rc);
        }
    }
    Py_RETURN_FALSE;
}

/* kv8_attend(scratch entry, entry, handle, 9 of the cache, 5 of the sequences, qt, q, qs, T, most, longest, Hq, out, scratch, win, scale, acc0, acc1) */
static PyObject *fast_kv8_attend(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    void *fs, *f, *g;
    kv8_t c;
    seqs_t s;
    buf_t q, out, sc, acc0, acc1;
    int64_t qt, qs, T, most, longest, Hq, win;
    float scale;
    if (n == 30 && get_address(a[0], &fs) && get_address(a[1], &f) && get_address(a[2], &g) && get_kv8(a + 3, &c) && get_seqs(a + 12, &s) && get_size(a[17], &qt) &&
        get_buf(a[18], &q) && get_size(a[19], &qs) && get_size(a[20], &T) && get_size(a[21], &most) && get_size(a[22], &longest) && get_size(a[23], &Hq) &&
        get_buf(a[24], &out) && get_opt(a[25], &sc) && get_size(a[26], &win) && get_float(a[27], &scale) && get_opt(a[28], &acc0) && get_opt(a[29], &acc1)) {
        const int64_t e = elt(qt);
        const __int128 acc = (__int128) c.blocks * c.Hkv * c.block * 4;
        if (e > 0 && T > 0 && Hq <= 1 << 20 && holds(&q, T, qs, Hq * c.D, e) && holds3(&out, T * e, Hq, c.D) && fits(&acc0, acc) && fits(&acc1, acc)) {
            __typeof__(&ns_kv8_attend_scratch) scratch = (__typeof__(&ns_kv8_attend_scratch)) fs;
            __typeof__(&ns_kv8_attend) call = (__typeof__(&ns_kv8_attend)) f;
            int rc = 0, room;
            Py_BEGIN_ALLOW_THREADS
            const int64_t need = scratch(s.S, most, Hq, c.Hkv, c.D, longest, acc1.ptr != NULL);
            room = need == 0 || (sc.ptr && fits(&sc, (__int128) need * 4));
            if (room)
                rc = call((ns_gpu *) g, (int) c.form, (int) qt, q.ptr, qs, T, (const int32_t *) s.start.ptr, (const int32_t *) s.lens.ptr, s.S, most, longest,
                          (const int32_t *) s.table.ptr, s.tmax, Hq, c.Hkv, c.D, c.block, c.blocks, c.k.ptr, c.v.ptr, (const float *) c.ks.ptr, (const float *) c.vs.ptr,
                          win, scale, out.ptr, (const float *) acc0.ptr, (float *) acc1.ptr, (float *) sc.ptr);
            Py_END_ALLOW_THREADS
            if (room) return made(rc);
        }
    }
    Py_RETURN_FALSE;
}

static PyMethodDef methods[] = {{"decode", (PyCFunction) (void (*)(void)) fast_decode, METH_FASTCALL, "attn.Ops.decode's checks and call"},
                                {"prompt", (PyCFunction) (void (*)(void)) fast_prompt, METH_FASTCALL, "attn.Ops.prompt's checks and call"},
                                {"pre_store", (PyCFunction) (void (*)(void)) fast_pre_store, METH_FASTCALL, "attn.Ops.pre_store's checks and call"},
                                {"norm_gated", (PyCFunction) (void (*)(void)) fast_norm_gated, METH_FASTCALL, "attn.Ops.norm_gated's checks and call"},
                                {"norm_residual", (PyCFunction) (void (*)(void)) fast_norm_residual, METH_FASTCALL, "attn.Ops.norm_residual's checks and call"},
                                {"q4_product", (PyCFunction) (void (*)(void)) fast_q4_product, METH_FASTCALL, "attn.Ops.q4_product's checks and call"},
                                {"ssm_step", (PyCFunction) (void (*)(void)) fast_ssm_step, METH_FASTCALL, "attn.Ops.ssm_step's checks and call"},
                                {"kv8_store", (PyCFunction) (void (*)(void)) fast_kv8_store, METH_FASTCALL, "attn.Ops.kv8_store's checks and call"},
                                {"kv8_attend", (PyCFunction) (void (*)(void)) fast_kv8_attend, METH_FASTCALL, "attn.Ops.kv8_attend's checks and call"},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops_fast", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__ops_fast(void) {
    s_ptr = PyUnicode_InternFromString("ptr");
    s_len = PyUnicode_InternFromString("len");
    return s_ptr && s_len ? PyModule_Create(&module) : NULL;
}
