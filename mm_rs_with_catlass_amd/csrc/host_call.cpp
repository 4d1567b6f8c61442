// The ordinary call of an operator from Python, without the Python: operands checked, descriptor filled in, launcher called.
//
// A call of a small launch is bound by what it does on the host (16x1024x8192 bf16 all-reduce of eight ranks: 6 to 7.5 us on the GPU, 10.8 us per
// call through Python and ctypes, of which the launch itself is 2.9).  call() takes the arguments of one operator call, and either launches
// it or returns None without having done anything: it accepts only what it has checked to the last condition the Python path
// checks, and everything else -- subclasses, wrapped tensors, numbers that are no Python integers, and all that is wrong -- goes through
// that path, which also says what is wrong.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string.h>

#include "catcoc_hip.h"

namespace {

// Addresses of the library the package has loaded (a second copy would have error state of its own).
decltype(&catcoc_get_kernel) getKernel;
decltype(&catcoc_launch_quant_matmul_reduce_scatter) launchQuant;
decltype(&catcoc_get_task_count) getTaskCount;
decltype(&catcoc_default_tiling) defaultTiling;
decltype(&catcoc_last_status) lastStatus;
decltype(&catcoc_last_error) lastError;
PyObject *errorType, *tilingType;   // CatcocError, CocTilingParams

PyObject *attach(PyObject *, PyObject *const *v, Py_ssize_t n)
{
    if (n != 8) return PyErr_Format(PyExc_TypeError, "attach takes six addresses and two types");
    void *p[6];
    for (int i = 0; i < 6; ++i) {
        p[i] = PyLong_AsVoidPtr(v[i]);
        if (p[i] == nullptr) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "address %d is null", i);
    }
    getKernel = (decltype(getKernel))p[0];
    launchQuant = (decltype(launchQuant))p[1];
    getTaskCount = (decltype(getTaskCount))p[2];
    defaultTiling = (decltype(defaultTiling))p[3];
    lastStatus = (decltype(lastStatus))p[4];
    lastError = (decltype(lastError))p[5];
    Py_INCREF(v[6]);
    Py_INCREF(v[7]);
    Py_XDECREF(errorType);
    Py_XDECREF(tilingType);
    errorType = v[6];
    tilingType = v[7];
    Py_RETURN_NONE;
}

// The arguments of call(), in order.  KIND is the CocCommType, or DECODE: the W8A8 operator with explicit kept rows.
enum { KIND, A, B, SCALE_A, SCALE_B, BIAS, PEERS, RANK, RANKS, TILING, TRANS_A, TRANS_B, PEER_ROW, FLAGS, OUTBOUND, CHECKSUM, DUMP, ACCUM, WORKSPACE, OUT,
       OUT_DTYPE, BLOCK_NUM, STAGES, SWIZZLE, SPLIT_K, KEPT_BEGIN, KEPT_ROWS, N0, ARGS };
constexpr int64_t DECODE = 4;

struct Other {};   // a call for the Python path

int64_t number(PyObject *o, int64_t hi = 0xffffffffll)
{
    if (!PyLong_Check(o)) throw Other{};
    int over = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &over);
    if (over || v < 0 || v > hi) throw Other{};
    return v;
}

// A plain tensor on the GPU without gaps, of the given type (Undefined: any) and dimensions (0: any).
const at::Tensor &tensor(PyObject *o, at::ScalarType type, int64_t dims, int64_t atLeast = 0)
{
    if (!THPVariable_CheckExact(o)) throw Other{};
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || !t.is_contiguous() || !t.has_storage() || (type != at::ScalarType::Undefined && t.scalar_type() != type) || (dims && t.dim() != dims) ||
        t.numel() < atLeast)
        throw Other{};
    return t;
}

uint8_t *address(const at::Tensor &t) { return (uint8_t *)t.mutable_data_ptr(); }

uint8_t *optional(PyObject *o, at::ScalarType type, int64_t dims, int64_t atLeast) { return o == Py_None ? nullptr : address(tensor(o, type, dims, atLeast)); }

PyObject *launch(PyObject *const *v)
{
    const int64_t kind = number(v[KIND], DECODE);
    const bool quant = kind >= QUANT_MATMUL_REDUCE_SCATTER, decode = kind == DECODE;
    const int comm = decode ? QUANT_MATMUL_REDUCE_SCATTER : (int)kind;
    const at::Tensor &a = tensor(v[A], quant ? at::kChar : at::ScalarType::Undefined, 2), &b = tensor(v[B], a.scalar_type(), 2);
    if (!quant && a.scalar_type() != at::kHalf && a.scalar_type() != at::kBFloat16) throw Other{};
    const int64_t P = number(v[RANKS], CATCOC_MAX_RANKS), rank = number(v[RANK], P - 1);   // (no rank: nothing is in range)
    const bool transA = number(v[TRANS_A], 1) != 0, transB = number(v[TRANS_B], 1) != 0;
    const int64_t m = a.size(transA ? 1 : 0), k = a.size(transA ? 0 : 1), n = b.size(transB ? 0 : 1);
    if (b.size(transB ? 1 : 0) != k || m > 0x7fffffff || k > 0x7fffffff || n > 0x7fffffff) throw Other{};
    const int64_t peerRow = number(v[PEER_ROW], 0x7fffffff);

    CatcocSymmetricDesc d{};
    d.magic = CATCOC_DESC_MAGIC;
    d.rankIdx = (uint32_t)rank;
    d.rankSize = (uint32_t)P;
    d.flags = (uint32_t)number(v[FLAGS]);
    d.blockNum = (uint32_t)number(v[BLOCK_NUM]);
    d.workspaceStages = (uint32_t)number(v[STAGES]);
    d.splitK = (uint32_t)number(v[SPLIT_K]);
    if (v[SWIZZLE] != Py_None) {
        if (!PyTuple_CheckExact(v[SWIZZLE]) || PyTuple_GET_SIZE(v[SWIZZLE]) != 2) throw Other{};
        d.swizzleOffset = (uint32_t)number(PyTuple_GET_ITEM(v[SWIZZLE], 0));
        d.swizzleDirection = (uint32_t)number(PyTuple_GET_ITEM(v[SWIZZLE], 1));
    }
    // ---- rows that are kept and written
    int64_t rows;
    if (decode) {
        const int64_t begin = number(v[KEPT_BEGIN]);
        rows = v[KEPT_ROWS] == Py_None ? m : number(v[KEPT_ROWS]);
        if (rows < 1 || begin + rows > m) throw Other{};
        d.keptRowBegin = (uint32_t)begin;
        d.keptRows = (uint32_t)rows;
    } else if (comm == MATMUL_ALLREDUCE) {
        rows = m;
    } else if (comm == ALLGATHER_MATMUL) {
        rows = m * P;
    } else {
        if (m % P != 0) throw Other{};
        rows = m / P;
    }
    // ---- peers
    const bool list = PyList_CheckExact(v[PEERS]);
    if (!list && !PyTuple_CheckExact(v[PEERS])) throw Other{};
    const Py_ssize_t peers = list ? PyList_GET_SIZE(v[PEERS]) : PyTuple_GET_SIZE(v[PEERS]);
    if (peers != P - 1) throw Other{};
    const at::ScalarType peerType = comm == ALLGATHER_MATMUL ? a.scalar_type() : quant && (d.flags & CATCOC_FLAG_REDUCE_INT32) ? at::kInt : at::kFloat;
    for (Py_ssize_t i = 0; i < peers; ++i) {
        const at::Tensor &p = tensor(list ? PyList_GET_ITEM(v[PEERS], i) : PyTuple_GET_ITEM(v[PEERS], i), peerType, 2);
        if (comm == ALLGATHER_MATMUL ? p.size(0) != m || p.size(1) != k : p.size(0) < peerRow + rows || p.size(1) < n || (i && p.size(1) != d.peerLd)) throw Other{};
        d.peers[i] = address(p);
        d.peerLd = p.size(1);
    }
    d.peerRowOffset = peerRow;
    // ---- the W8A8 operator's vectors, and what both kinds may be given
    uint8_t *scaleA = nullptr, *scaleB = nullptr, *bias = nullptr, *accum = nullptr;
    if (quant) {
        scaleA = address(tensor(v[SCALE_A], at::kFloat, 1, m));
        scaleB = address(tensor(v[SCALE_B], at::kFloat, 1, n));
        bias = optional(v[BIAS], at::kInt, 1, n);
        accum = optional(v[ACCUM], at::kInt, 0, rows * n);
    }
    d.accDump = optional(v[DUMP], quant ? at::kInt : at::kFloat, 0, (comm == ALLGATHER_MATMUL ? rows : m) * n);
    if (v[OUTBOUND] != Py_None) {
        const at::Tensor &t = tensor(v[OUTBOUND], at::ScalarType::Undefined, 0);
        if (t.scalar_type() != at::kFloat && !(quant && t.scalar_type() == at::kInt)) throw Other{};
        d.outbound = address(t);
        d.outboundBytes = (uint64_t)t.nbytes();
    }
    if (v[WORKSPACE] != Py_None) {
        const at::Tensor &t = tensor(v[WORKSPACE], at::ScalarType::Undefined, 0);
        d.workspace = address(t);
        d.workspaceBytes = (uint64_t)t.nbytes();
    }
    // ---- tiling: the caller's, or the library's tiles
    CocTilingParams tiling;
    if (v[TILING] == Py_None) {
        const int64_t n0 = number(v[N0]);
        defaultTiling(&tiling, (uint32_t)m, (uint32_t)k, (uint32_t)n, (uint32_t)P);
        tiling.commInterval = 1;
        tiling.m0 = n0 ? 128 : 0;
        tiling.n0 = (uint32_t)n0;
        tiling.k0 = 0;
    } else {
        Py_buffer view;
        if ((PyObject *)Py_TYPE(v[TILING]) != tilingType || PyObject_GetBuffer(v[TILING], &view, PyBUF_SIMPLE) != 0) {
            PyErr_Clear();
            throw Other{};
        }
        memcpy(&tiling, view.buf, sizeof tiling);
        PyBuffer_Release(&view);
        if (tiling.m != m || tiling.k != k || tiling.n != n) throw Other{};
    }
    if (v[CHECKSUM] != Py_None) {
        int64_t need;
        if (decode) {
            need = (m + 127) / 128 * ((n + 127) / 128);
        } else {
            need = getTaskCount(comm, &tiling, &d);
            if (lastStatus() != 0) throw Other{};
        }
        d.checksum = (int64_t *)address(tensor(v[CHECKSUM], quant ? at::kLong : at::kDouble, 0, need));
    }
    // ---- output
    at::Tensor made;
    const at::Tensor *out = &made;
    if (v[OUT] != Py_None) {
        out = &tensor(v[OUT], quant ? at::ScalarType::Undefined : a.scalar_type(), 2);
        if ((out->scalar_type() != at::kHalf && out->scalar_type() != at::kBFloat16) || out->size(0) != rows || out->size(1) != n) throw Other{};
    } else {
        at::ScalarType type = a.scalar_type();
        if (quant) {
            if (!THPDtype_Check(v[OUT_DTYPE])) throw Other{};
            type = ((THPDtype *)v[OUT_DTYPE])->scalar_type;
            if (type != at::kHalf && type != at::kBFloat16) throw Other{};
        }
        made = at::empty({rows, n}, a.options().dtype(type));
    }
    uint8_t *const pa = address(a), *const pb = address(b), *const po = address(*out);
    const uint32_t outType = out->scalar_type() == at::kHalf ? FP16 : BF16;
    void *const stream = (void *)c10::hip::getCurrentHIPStream().stream();
    const auto kernel = quant ? nullptr : getKernel(comm, (int)outType);
    if (!quant && kernel == nullptr) throw Other{};
    Py_BEGIN_ALLOW_THREADS
    if (quant) launchQuant(stream, 0, pa, pb, scaleA, scaleB, bias, accum, po, (uint8_t *)&d, &tiling, transA, transB, outType);
    else kernel(stream, 0, pa, pb, po, nullptr, nullptr, (uint8_t *)&d, &tiling, transA, transB);
    Py_END_ALLOW_THREADS
    if (lastStatus() != 0) {
        PyErr_SetString(errorType, lastError());
        return nullptr;
    }
    if (v[OUT] == Py_None) return THPVariable_Wrap(std::move(made));
    Py_INCREF(v[OUT]);
    return v[OUT];
}

PyObject *call(PyObject *, PyObject *const *v, Py_ssize_t n)
{
    if (n != ARGS || errorType == nullptr) return PyErr_Format(PyExc_TypeError, "call takes %d arguments, after attach", (int)ARGS);
    try {
        return launch(v);
    } catch (const Other &) {
    } catch (const std::exception &) {   // (a tensor without memory of its own, no memory for the output: the Python path meets it again)
        PyErr_Clear();
    }
    Py_RETURN_NONE;
}

// ---- e4m3 and grouped operators: quantize_fp8() and its like below, of the same kind as call().
decltype(&catcoc_quantize_fp8) quantizeFp8;
decltype(&catcoc_fp8_matmul_allreduce) fp8Matmul;
decltype(&catcoc_grouped_matmul) groupedMatmul;
decltype(&catcoc_grouped_matmul_dw) groupedDw;
decltype(&catcoc_grouped_fp8_matmul) groupedFp8;

PyObject *attachRagged(PyObject *, PyObject *const *v, Py_ssize_t n)
{
    if (n != 5) return PyErr_Format(PyExc_TypeError, "attach_ragged takes five addresses");
    void *p[5];
    for (int i = 0; i < 5; ++i) {
        p[i] = PyLong_AsVoidPtr(v[i]);
        if (p[i] == nullptr) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "address %d is null", i);
    }
    quantizeFp8 = (decltype(quantizeFp8))p[0];
    fp8Matmul = (decltype(fp8Matmul))p[1];
    groupedMatmul = (decltype(groupedMatmul))p[2];
    groupedDw = (decltype(groupedDw))p[3];
    groupedFp8 = (decltype(groupedFp8))p[4];
    Py_RETURN_NONE;
}

constexpr int64_t BLOCK = 128, MOST = 0x7fffffff;
constexpr at::ScalarType F8 = at::ScalarType::Float8_e4m3fn;

int64_t blocks(int64_t n) { return (n + BLOCK - 1) / BLOCK; }

// A tensor of exactly this shape, or, None, a new one.
struct Result {
    at::Tensor made;
    const at::Tensor *t = &made;
    PyObject *given = nullptr;

    Result(PyObject *o, at::ScalarType type, at::IntArrayRef shape, const at::Tensor &like)
    {
        if (o == Py_None) {
            made = at::empty(shape, like.options().dtype(type));
            return;
        }
        t = &tensor(o, type, (int64_t)shape.size());
        if (t->sizes() != shape) throw Other{};
        given = o;
    }
    Result(const Result &) = delete;
    uint8_t *at_() { return address(*t); }
    PyObject *object()
    {
        if (given == nullptr) return THPVariable_Wrap(std::move(made));
        Py_INCREF(given);
        return given;
    }
};

const at::Tensor &shaped(PyObject *o, at::ScalarType type, at::IntArrayRef shape)
{
    const at::Tensor &t = tensor(o, type, (int64_t)shape.size());
    if (t.sizes() != shape) throw Other{};
    return t;
}

uint32_t code(at::ScalarType t, bool floats = false)
{
    if (t == at::kHalf) return FP16;
    if (t == at::kBFloat16) return BF16;
    if (floats && t == at::kFloat) return 0;
    throw Other{};
}

// The type of a result: that of `out`, else what is asked for.
at::ScalarType resultType(PyObject *out, PyObject *dtype)
{
    if (out != Py_None) return THPVariable_CheckExact(out) ? THPVariable_Unpack(out).scalar_type() : throw Other{};
    if (!THPDtype_Check(dtype)) throw Other{};
    return ((THPDtype *)dtype)->scalar_type;
}

void *stream() { return (void *)c10::hip::getCurrentHIPStream().stream(); }

template <typename F>
PyObject *guarded(const char *name, Py_ssize_t n, Py_ssize_t wanted, F &&body)
{
    if (n != wanted || errorType == nullptr || groupedFp8 == nullptr) return PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, after attach and attach_ragged", name, wanted);
    try {
        return body();
    } catch (const Other &) {
    } catch (const std::exception &) {
        PyErr_Clear();
    }
    Py_RETURN_NONE;
}

// What the library answered: false where it refused (the error is set).
bool accepted()
{
    if (lastStatus() == 0) return true;
    PyErr_SetString(errorType, lastError());
    return false;
}

PyObject *quantize(PyObject *, PyObject *const *v, Py_ssize_t n)   // x, block_rows, gated, out, scale
{
    return guarded("quantize_fp8", n, 5, [&]() -> PyObject * {
        const at::Tensor &x = tensor(v[0], at::ScalarType::Undefined, 2);
        const uint32_t type = code(x.scalar_type(), true);
        const int64_t blockRows = number(v[1], BLOCK);
        const bool gated = number(v[2], 1) != 0;
        const int64_t rows = x.size(0), cols = gated ? x.size(1) / 2 : x.size(1);
        if ((blockRows != 1 && blockRows != BLOCK) || (gated && (blockRows != 1 || x.size(1) % 2 != 0)) || rows > MOST || cols > MOST) throw Other{};
        Result q(v[3], F8, {rows, cols}, x);
        Result scale(v[4], at::kFloat, blockRows == 1 ? at::IntArrayRef({blocks(cols), rows}) : at::IntArrayRef({blocks(rows), blocks(cols)}), x);
        uint8_t *const px = address(x), *const pq = q.at_();
        float *const ps = (float *)scale.at_();
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        quantizeFp8(s, px, pq, ps, (uint32_t)rows, (uint32_t)cols, (uint32_t)blockRows, gated, type);
        Py_END_ALLOW_THREADS
        if (!accepted()) return nullptr;
        PyObject *a = q.object(), *b = scale.object(), *both = a && b ? PyTuple_Pack(2, a, b) : nullptr;
        Py_XDECREF(a);
        Py_XDECREF(b);
        return both;
    });
}

PyObject *fp8(PyObject *, PyObject *const *v, Py_ssize_t n)   // x1, x2, scale_x1, scale_x2, peers, rank, rank_size, out_dtype, peer_row_offset, out
{
    return guarded("fp8_matmul_allreduce", n, 10, [&]() -> PyObject * {
        const at::Tensor &x = tensor(v[0], F8, 2), &w = tensor(v[1], F8, 2);
        const int64_t m = x.size(0), k = x.size(1), cols = w.size(0);
        if (w.size(1) != k || m > MOST || k > MOST || cols > MOST) throw Other{};
        const at::Tensor &sx = shaped(v[2], at::kFloat, {blocks(k), m}), &sw = shaped(v[3], at::kFloat, {blocks(cols), blocks(k)});
        const int64_t P = number(v[6], CATCOC_MAX_RANKS), rank = number(v[5], P - 1), peerRow = number(v[8], MOST);
        const bool list = PyList_CheckExact(v[4]);
        if ((!list && !PyTuple_CheckExact(v[4])) || (list ? PyList_GET_SIZE(v[4]) : PyTuple_GET_SIZE(v[4])) != P - 1) throw Other{};
        CatcocSymmetricDesc d{};
        d.magic = CATCOC_DESC_MAGIC;
        d.rankIdx = (uint32_t)rank;
        d.rankSize = (uint32_t)P;
        d.peerRowOffset = peerRow;
        for (Py_ssize_t i = 0; i < P - 1; ++i) {
            const at::Tensor &p = tensor(list ? PyList_GET_ITEM(v[4], i) : PyTuple_GET_ITEM(v[4], i), at::kFloat, 2);
            if (p.size(0) < peerRow + m || p.size(1) < cols || (i && p.size(1) != d.peerLd)) throw Other{};
            d.peers[i] = address(p);
            d.peerLd = p.size(1);
        }
        const at::ScalarType type = resultType(v[9], v[7]);
        const uint32_t outType = code(type);
        Result out(v[9], type, {m, cols}, x);
        uint8_t *const px = address(x), *const pw = address(w), *const po = out.at_();
        const float *const psx = (const float *)address(sx), *const psw = (const float *)address(sw);
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        fp8Matmul(s, px, pw, psx, psw, po, (uint8_t *)&d, (uint32_t)m, (uint32_t)cols, (uint32_t)k, outType, nullptr);
        Py_END_ALLOW_THREADS
        return accepted() ? out.object() : nullptr;
    });
}

PyObject *grouped(PyObject *, PyObject *const *v, Py_ssize_t n)   // x, w, group_ends, trans_b, out
{
    return guarded("grouped_matmul", n, 5, [&]() -> PyObject * {
        const at::Tensor &x = tensor(v[0], at::ScalarType::Undefined, 2);
        const uint32_t type = code(x.scalar_type());
        const at::Tensor &w = tensor(v[1], x.scalar_type(), 3);
        const bool transB = number(v[3], 1) != 0;
        const int64_t rows = x.size(0), k = x.size(1), groups = w.size(0), cols = w.size(transB ? 1 : 2);
        if (w.size(transB ? 2 : 1) != k || rows > MOST || k > MOST || cols > MOST || groups < 1 || groups > MOST) throw Other{};
        const int32_t *const ends = (const int32_t *)address(shaped(v[2], at::kInt, {groups}));
        Result out(v[4], x.scalar_type(), {rows, cols}, x);
        uint8_t *const px = address(x), *const pw = address(w), *const po = out.at_();
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        groupedMatmul(s, type, px, pw, ends, po, (uint32_t)rows, (uint32_t)cols, (uint32_t)k, (uint32_t)groups, transB, nullptr);
        Py_END_ALLOW_THREADS
        return accepted() ? out.object() : nullptr;
    });
}

PyObject *dw(PyObject *, PyObject *const *v, Py_ssize_t n)   // x, dy, group_ends, out_dtype, trans_b, out
{
    return guarded("grouped_matmul_dw", n, 6, [&]() -> PyObject * {
        const at::Tensor &x = tensor(v[0], at::ScalarType::Undefined, 2);
        const uint32_t type = code(x.scalar_type());
        const at::Tensor &dy = tensor(v[1], x.scalar_type(), 2), &e = tensor(v[2], at::kInt, 1);
        const bool transB = number(v[4], 1) != 0;
        const int64_t rows = x.size(0), k = x.size(1), groups = e.size(0), cols = dy.size(1);
        if (dy.size(0) != rows || rows > MOST || k > MOST || cols > MOST || groups < 1 || groups > MOST) throw Other{};
        const at::ScalarType made = v[5] == Py_None && v[3] == Py_None ? x.scalar_type() : resultType(v[5], v[3]);
        const uint32_t outType = code(made, true);
        Result out(v[5], made, transB ? at::IntArrayRef({groups, cols, k}) : at::IntArrayRef({groups, k, cols}), x);
        uint8_t *const px = address(x), *const pd = address(dy), *const po = out.at_();
        const int32_t *const ends = (const int32_t *)address(e);
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        groupedDw(s, type, px, pd, ends, po, (uint32_t)rows, (uint32_t)cols, (uint32_t)k, (uint32_t)groups, transB, outType, nullptr);
        Py_END_ALLOW_THREADS
        return accepted() ? out.object() : nullptr;
    });
}

PyObject *fp8Grouped(PyObject *, PyObject *const *v, Py_ssize_t n)   // x, w, scale_x, scale_w, group_ends, out_dtype, out
{
    return guarded("grouped_fp8_matmul", n, 7, [&]() -> PyObject * {
        const at::Tensor &x = tensor(v[0], F8, 2), &w = tensor(v[1], F8, 3);
        const int64_t rows = x.size(0), k = x.size(1), groups = w.size(0), cols = w.size(1);
        if (w.size(2) != k || rows > MOST || k > MOST || cols > MOST || groups < 1 || groups > MOST) throw Other{};
        const at::Tensor &sx = shaped(v[2], at::kFloat, {blocks(k), rows}), &sw = shaped(v[3], at::kFloat, {groups, blocks(cols), blocks(k)});
        const int32_t *const ends = (const int32_t *)address(shaped(v[4], at::kInt, {groups}));
        const at::ScalarType type = resultType(v[6], v[5]);
        const uint32_t outType = code(type);
        Result out(v[6], type, {rows, cols}, x);
        uint8_t *const px = address(x), *const pw = address(w), *const po = out.at_();
        const float *const psx = (const float *)address(sx), *const psw = (const float *)address(sw);
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        groupedFp8(s, px, pw, psx, psw, ends, po, (uint32_t)rows, (uint32_t)cols, (uint32_t)k, (uint32_t)groups, outType, nullptr);
        Py_END_ALLOW_THREADS
        return accepted() ? out.object() : nullptr;
    });
}

PyMethodDef methods[] = {{"attach_ragged", (PyCFunction)(void *)attachRagged, METH_FASTCALL, "addresses of the e4m3 and grouped operators' functions"},
                         {"quantize_fp8", (PyCFunction)(void *)quantize, METH_FASTCALL, "one call: (codes, scale), or None for the Python path"},
                         {"fp8_matmul_allreduce", (PyCFunction)(void *)fp8, METH_FASTCALL, "one call: the output, or None for the Python path"},
                         {"grouped_matmul", (PyCFunction)(void *)grouped, METH_FASTCALL, "one call: the output, or None for the Python path"},
                         {"grouped_matmul_dw", (PyCFunction)(void *)dw, METH_FASTCALL, "one call: the output, or None for the Python path"},
                         {"grouped_fp8_matmul", (PyCFunction)(void *)fp8Grouped, METH_FASTCALL, "one call: the output, or None for the Python path"},
                         {"attach", (PyCFunction)(void *)attach, METH_FASTCALL, "addresses of the library's functions, CatcocError, CocTilingParams"},
                         {"call", (PyCFunction)(void *)call, METH_FASTCALL, "one operator call: the output, or None for the Python path"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
