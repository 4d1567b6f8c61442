// The ordinary call of an operator from Python, without the Python: operands checked, descriptor filled in, launcher called.
//
// A call of a small launch is bound by what it does on the host (16x1024x8192 bf16 all-reduce of eight ranks: 6 to 7.5 us on the GPU, 10.8 us per
// call through Python and ctypes, of which the launch itself is 2.9).  call() takes the arguments of one operator call, and either launches
// it or returns None without having done anything: it accepts only what it has checked to the last condition the Python path
// checks, and everything else -- subclasses, wrapped tensors, numbers that are no Python integers, and all that is wrong -- goes through
// that path, which also says what is wrong.
#include <Python.h>

#include <ATen/Context.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string.h>

#include <initializer_list>
#include <optional>

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

// A new tensor, made without the dispatcher's two turns (0.25 us of a call's 4 to 6.4 for each output), unless there is a mode that they serve: a dispatch mode, which
// sees what is made, or the deterministic one, which fills it.
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const at::Tensor &like)
{
    const at::Context &context = at::globalContext();
    if (c10::impl::TorchDispatchModeTLS::any_modes_set() || (context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory()))
        return at::empty(shape, like.options().dtype(type));
    return at::Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}

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
        made = fresh({rows, n}, type, a);
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
            made = fresh(shape, type, like);
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

// ---- operators around a layer of experts: rms_norm() and those below it in ops.py, of the same kind.
decltype(&catcoc_rms_norm) rmsNorm;
decltype(&catcoc_rms_norm_backward) rmsNormBackward;
decltype(&catcoc_rms_norm_backward_workspace_size) rmsNormWorkspace;
decltype(&catcoc_route) routeTo;
decltype(&catcoc_route_backward) routeBackward;
decltype(&catcoc_sort_by_expert) sortByExpert;
decltype(&catcoc_sort_by_expert_workspace_size) sortWorkspace;
decltype(&catcoc_spread_rows) spreadRows;
decltype(&catcoc_gather_rows) gatherRows;
decltype(&catcoc_gather_rows_backward) gatherBackward;

PyObject *attachLayer(PyObject *, PyObject *const *v, Py_ssize_t n)
{
    if (n != 10) return PyErr_Format(PyExc_TypeError, "attach_layer takes ten addresses");
    void *p[10];
    for (int i = 0; i < 10; ++i) {
        p[i] = PyLong_AsVoidPtr(v[i]);
        if (p[i] == nullptr) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "address %d is null", i);
    }
    rmsNorm = (decltype(rmsNorm))p[0];
    rmsNormBackward = (decltype(rmsNormBackward))p[1];
    rmsNormWorkspace = (decltype(rmsNormWorkspace))p[2];
    routeTo = (decltype(routeTo))p[3];
    routeBackward = (decltype(routeBackward))p[4];
    sortByExpert = (decltype(sortByExpert))p[5];
    sortWorkspace = (decltype(sortWorkspace))p[6];
    spreadRows = (decltype(spreadRows))p[7];
    gatherRows = (decltype(gatherRows))p[8];
    gatherBackward = (decltype(gatherBackward))p[9];
    Py_RETURN_NONE;
}

// Tensors on the current device, whose stream the call goes to.
struct Here {
    const c10::DeviceIndex device = c10::hip::current_device();

    const at::Tensor &any(PyObject *o, int64_t dims) const
    {
        const at::Tensor &t = tensor(o, at::ScalarType::Undefined, dims);
        if (t.get_device() != device) throw Other{};
        return t;
    }
    const at::Tensor &of(PyObject *o, at::ScalarType type, at::IntArrayRef shape) const
    {
        const at::Tensor &t = shaped(o, type, shape);
        if (t.get_device() != device) throw Other{};
        return t;
    }
    uint8_t *maybe(PyObject *o, at::ScalarType type, at::IntArrayRef shape) const { return o == Py_None ? nullptr : address(of(o, type, shape)); }
    void check(const Result &r) const
    {
        if (r.t->get_device() != device) throw Other{};
    }
};

// The type of an operand that is of type `own` or fp32.
at::ScalarType likeOrWide(PyObject *o, at::ScalarType own)
{
    if (!THPVariable_CheckExact(o)) throw Other{};
    const at::ScalarType t = THPVariable_Unpack(o).scalar_type();
    if (t != own && t != at::kFloat) throw Other{};
    return t;
}

double real(PyObject *o)
{
    if (!PyFloat_CheckExact(o)) throw Other{};
    return PyFloat_AS_DOUBLE(o);
}

template <typename F>
PyObject *guardedLayer(const char *name, Py_ssize_t n, Py_ssize_t wanted, F &&body)
{
    if (gatherBackward == nullptr) return PyErr_Format(PyExc_TypeError, "%s comes after attach_layer", name);
    return guarded(name, n, wanted, body);
}

PyObject *tupleOf(std::initializer_list<Result *> results)
{
    PyObject *all = PyTuple_New((Py_ssize_t)results.size());
    Py_ssize_t i = 0;
    for (Result *r : results) {
        PyObject *o = all ? r->object() : nullptr;
        if (o == nullptr) {
            Py_XDECREF(all);
            return nullptr;
        }
        PyTuple_SET_ITEM(all, i++, o);
    }
    return all;
}

// Both norms: x, weight, residual, eps, then for the first out, residual_out; for the second keep, out, scale, kept, residual_out.
PyObject *norm(PyObject *const *v, bool fp8)
{
    const Here here;
    const at::Tensor &x = here.any(v[0], 2);
    const int64_t rows = x.size(0), cols = x.size(1);
    const at::ScalarType type = x.scalar_type(), weightType = likeOrWide(v[1], type);
    const uint32_t typeCode = code(type, true);
    if (rows > MOST || cols > MOST) throw Other{};
    const int64_t sizes[2] = {rows, cols};
    const at::IntArrayRef shape(sizes, 2);
    const at::Tensor &weight = here.of(v[1], weightType, {cols});
    const bool summed = v[2] != Py_None, keep = !fp8 || number(v[4], 1) != 0;
    PyObject *const out = v[fp8 ? 7 : 4], *const sumOut = v[fp8 ? 8 : 5];
    if ((!summed && sumOut != Py_None) || (!keep && out != Py_None)) throw Other{};
    const at::ScalarType sumType = summed ? likeOrWide(v[2], type) : type;
    uint8_t *const residual = here.maybe(v[2], sumType, shape);
    const float eps = (float)real(v[3]);
    std::optional<Result> y, sum, q, scale;
    if (keep) here.check(y.emplace(out, type, shape, x));
    if (summed) here.check(sum.emplace(sumOut, sumType, shape, x));
    if (fp8) {
        here.check(q.emplace(v[5], F8, shape, x));
        here.check(scale.emplace(v[6], at::kFloat, at::IntArrayRef({blocks(cols), rows}), x));
    }
    uint8_t *const px = address(x), *const pw = address(weight), *const py = y ? y->at_() : nullptr, *const ps = sum ? sum->at_() : nullptr;
    uint8_t *const pq = q ? q->at_() : nullptr;
    float *const pscale = scale ? (float *)scale->at_() : nullptr;
    const uint32_t sumCode = code(sumType, true), weightCode = code(weightType, true);
    void *const s = stream();
    Py_BEGIN_ALLOW_THREADS
    rmsNorm(s, px, residual, pw, py, ps, pq, pscale, (uint32_t)rows, (uint32_t)cols, eps, typeCode, sumCode, weightCode);
    Py_END_ALLOW_THREADS
    if (!accepted()) return nullptr;
    if (!fp8) return summed ? tupleOf({&*y, &*sum}) : y->object();
    if (keep) return summed ? tupleOf({&*q, &*scale, &*y, &*sum}) : tupleOf({&*q, &*scale, &*y});
    return summed ? tupleOf({&*q, &*scale, &*sum}) : tupleOf({&*q, &*scale});
}

PyObject *norm16(PyObject *, PyObject *const *v, Py_ssize_t n)   // x, weight, residual, eps, out, residual_out
{
    return guardedLayer("rms_norm", n, 6, [&] { return norm(v, false); });
}

PyObject *normFp8(PyObject *, PyObject *const *v, Py_ssize_t n)   // x, weight, residual, eps, keep, out, scale, kept, residual_out
{
    return guardedLayer("rms_norm_fp8", n, 9, [&] { return norm(v, true); });
}

PyObject *normBackward(PyObject *, PyObject *const *v, Py_ssize_t n)   // dy, x, weight, dsum, eps, dx, dw
{
    return guardedLayer("rms_norm_backward", n, 7, [&]() -> PyObject * {
        const Here here;
        const at::Tensor &dy = here.any(v[0], 2);
        const int64_t rows = dy.size(0), cols = dy.size(1);
        const at::ScalarType type = dy.scalar_type(), sumType = likeOrWide(v[1], type), weightType = likeOrWide(v[2], type);
        const uint32_t typeCode = code(type, true), sumCode = code(sumType, true), weightCode = code(weightType, true);
        if (rows > MOST || cols > MOST) throw Other{};
        const int64_t sizes[2] = {rows, cols};
        const at::IntArrayRef shape(sizes, 2);
        const at::Tensor &x = here.of(v[1], sumType, shape), &weight = here.of(v[2], weightType, {cols});
        uint8_t *const dsum = here.maybe(v[3], sumType, shape);
        const float eps = (float)real(v[4]);
        Result dx(v[5], sumType, shape, x), dw(v[6], weightType, {cols}, x);
        here.check(dx);
        here.check(dw);
        const uint64_t bytes = rmsNormWorkspace((uint32_t)rows, (uint32_t)cols);
        const at::Tensor work = fresh({(int64_t)bytes}, at::kByte, x);
        uint8_t *const pd = address(dy), *const px = address(x), *const pw = address(weight), *const pdx = dx.at_(), *const pdw = dw.at_(), *const pwork = address(work);
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        rmsNormBackward(s, pd, px, pw, dsum, pdx, pdw, pwork, bytes, (uint32_t)rows, (uint32_t)cols, eps, typeCode, sumCode, weightCode);
        Py_END_ALLOW_THREADS
        return accepted() ? tupleOf({&dx, &dw}) : nullptr;
    });
}

uint32_t score(PyObject *o)
{
    if (!PyUnicode_CheckExact(o)) throw Other{};
    if (PyUnicode_CompareWithASCIIString(o, "softmax") == 0) return CATCOC_SCORE_SOFTMAX;
    if (PyUnicode_CompareWithASCIIString(o, "sigmoid") == 0) return CATCOC_SCORE_SIGMOID;
    throw Other{};
}

uint32_t positive(PyObject *o)
{
    const int64_t v = number(o, MOST);
    if (v < 1) throw Other{};
    return (uint32_t)v;
}

PyObject *route(PyObject *, PyObject *const *v, Py_ssize_t n)   // logits, top, score, bias, groups, top_groups, group_top, renormalize, scale, choice, share
{
    return guardedLayer("route", n, 11, [&]() -> PyObject * {
        const Here here;
        const at::Tensor &logits = here.any(v[0], 2);
        const int64_t tokens = logits.size(0), experts = logits.size(1), top = positive(v[1]);
        const uint32_t type = code(logits.scalar_type(), true);
        if (tokens > MOST || experts > MOST || top > experts) throw Other{};
        CatcocRouting how{score(v[2]), positive(v[4]), positive(v[5]), positive(v[6]), (uint32_t)number(v[7], 1), (float)real(v[8])};
        const float *const bias = (const float *)here.maybe(v[3], at::kFloat, {experts});
        Result choice(v[9], at::kInt, {tokens, top}, logits), share(v[10], at::kFloat, {tokens, top}, logits);
        here.check(choice);
        here.check(share);
        uint8_t *const px = address(logits);
        int32_t *const pc = (int32_t *)choice.at_();
        float *const ps = (float *)share.at_();
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        routeTo(s, px, bias, pc, ps, &how, (uint32_t)tokens, (uint32_t)experts, (uint32_t)top, type);
        Py_END_ALLOW_THREADS
        return accepted() ? tupleOf({&choice, &share}) : nullptr;
    });
}

PyObject *routeGradient(PyObject *, PyObject *const *v, Py_ssize_t n)   // dshare, logits, choice, score, renormalize, scale, out
{
    return guardedLayer("route_backward", n, 7, [&]() -> PyObject * {
        const Here here;
        const at::Tensor &logits = here.any(v[1], 2), &choice = here.any(v[2], 2);
        const int64_t tokens = logits.size(0), experts = logits.size(1), top = choice.size(1);
        const uint32_t type = code(logits.scalar_type(), true);
        if (choice.scalar_type() != at::kInt || choice.size(0) != tokens || tokens > MOST || experts > MOST || top > experts) throw Other{};
        const at::Tensor &dshare = here.of(v[0], at::kFloat, {tokens, top});
        CatcocRouting how{score(v[3]), 1, 1, 1, (uint32_t)number(v[4], 1), (float)real(v[5])};
        Result out(v[6], logits.scalar_type(), {tokens, experts}, logits);
        here.check(out);
        uint8_t *const px = address(logits), *const po = out.at_();
        const float *const pd = (const float *)address(dshare);
        const int32_t *const pc = (const int32_t *)address(choice);
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        routeBackward(s, pd, px, pc, po, &how, (uint32_t)tokens, (uint32_t)experts, (uint32_t)top, type);
        Py_END_ALLOW_THREADS
        return accepted() ? out.object() : nullptr;
    });
}

PyObject *sortChoices(PyObject *, PyObject *const *v, Py_ssize_t n)   // choice, experts, order, back, ends
{
    return guardedLayer("sort_by_expert", n, 5, [&]() -> PyObject * {
        const Here here;
        const at::Tensor &choice = here.any(v[0], 2);
        const int64_t rows = choice.numel(), experts = positive(v[1]);
        const bool wide = choice.scalar_type() == at::kLong;
        if ((!wide && choice.scalar_type() != at::kInt) || rows > MOST || experts > 1024) throw Other{};
        Result order(v[2], at::kInt, {rows}, choice), back(v[3], at::kInt, choice.sizes(), choice), ends(v[4], at::kInt, {experts}, choice);
        here.check(order);
        here.check(back);
        here.check(ends);
        const uint64_t bytes = sortWorkspace((uint32_t)rows, (uint32_t)experts);
        at::Tensor work;
        if (bytes) work = fresh({(int64_t)bytes}, at::kByte, choice);
        uint8_t *const pc = address(choice), *const pwork = bytes ? address(work) : nullptr;
        int32_t *const po = (int32_t *)order.at_(), *const pb = (int32_t *)back.at_(), *const pe = (int32_t *)ends.at_();
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        sortByExpert(s, pc, po, pb, pe, pwork, bytes, (uint32_t)rows, (uint32_t)experts, wide ? 64 : 32);
        Py_END_ALLOW_THREADS
        return accepted() ? tupleOf({&order, &back, &ends}) : nullptr;
    });
}

PyObject *spread(PyObject *, PyObject *const *v, Py_ssize_t n)   // x, back, scale, out, out_scale
{
    return guardedLayer("spread_rows", n, 5, [&]() -> PyObject * {
        const Here here;
        const at::Tensor &x = here.any(v[0], 2), &back = here.any(v[1], 2);
        const int64_t tokens = x.size(0), cols = x.size(1), top = back.size(1);
        if (x.scalar_type() != F8) code(x.scalar_type(), true);
        if (back.scalar_type() != at::kInt || back.size(0) != tokens || back.numel() > MOST || tokens > MOST || top > MOST || cols > MOST) throw Other{};
        const bool scaled = v[2] != Py_None;
        if (scaled ? x.scalar_type() != F8 : v[4] != Py_None) throw Other{};
        const float *const scale = (const float *)here.maybe(v[2], at::kFloat, {blocks(cols), tokens});
        Result out(v[3], x.scalar_type(), {tokens * top, cols}, x);
        here.check(out);
        std::optional<Result> outScale;
        if (scaled) here.check(outScale.emplace(v[4], at::kFloat, at::IntArrayRef({blocks(cols), tokens * top}), x));
        uint8_t *const px = address(x), *const po = out.at_();
        const int32_t *const pb = (const int32_t *)address(back);
        float *const ps = scaled ? (float *)outScale->at_() : nullptr;
        const uint32_t size = (uint32_t)x.element_size();
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        spreadRows(s, px, scale, pb, po, ps, (uint32_t)tokens, (uint32_t)top, (uint32_t)cols, size);
        Py_END_ALLOW_THREADS
        if (!accepted()) return nullptr;
        return scaled ? tupleOf({&out, &*outScale}) : out.object();
    });
}

PyObject *gather(PyObject *, PyObject *const *v, Py_ssize_t n)   // y, back, share, out
{
    return guardedLayer("gather_rows", n, 4, [&]() -> PyObject * {
        const Here here;
        const at::Tensor &y = here.any(v[0], 2), &back = here.any(v[1], 2);
        const int64_t tokens = back.size(0), top = back.size(1), cols = y.size(1);
        const uint32_t type = code(y.scalar_type(), true);
        if (back.scalar_type() != at::kInt || y.size(0) != back.numel() || y.size(0) > MOST || tokens > MOST || top > MOST || cols > MOST) throw Other{};
        const float *const share = (const float *)here.maybe(v[2], at::kFloat, {tokens, top});
        Result out(v[3], y.scalar_type(), {tokens, cols}, y);
        here.check(out);
        uint8_t *const py = address(y), *const po = out.at_();
        const int32_t *const pb = (const int32_t *)address(back);
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        gatherRows(s, py, pb, share, po, (uint32_t)tokens, (uint32_t)top, (uint32_t)cols, type);
        Py_END_ALLOW_THREADS
        return accepted() ? out.object() : nullptr;
    });
}

PyObject *gatherGradient(PyObject *, PyObject *const *v, Py_ssize_t n)   // dout, y, back, share, dy, dshare, rows
{
    return guardedLayer("gather_rows_backward", n, 7, [&]() -> PyObject * {
        const Here here;
        const bool rows = number(v[6], 1) != 0, shares = v[1] != Py_None;
        if ((!rows && (!shares || v[4] != Py_None)) || (!shares && v[5] != Py_None)) throw Other{};
        const at::Tensor &dout = here.any(v[0], 2), &back = here.any(v[2], 2);
        const int64_t tokens = back.size(0), top = back.size(1), cols = dout.size(1);
        const at::ScalarType type = dout.scalar_type();
        const uint32_t typeCode = code(type, true);
        if (back.scalar_type() != at::kInt || dout.size(0) != tokens || back.numel() > MOST || tokens > MOST || top > MOST || cols > MOST) throw Other{};
        const int64_t sizes[2] = {tokens * top, cols};
        const at::IntArrayRef spread(sizes, 2);
        const at::Tensor &share = here.of(v[3], at::kFloat, {tokens, top});
        uint8_t *const py = here.maybe(v[1], type, spread);
        std::optional<Result> dy, dshare;
        if (rows) here.check(dy.emplace(v[4], type, spread, dout));
        if (shares) here.check(dshare.emplace(v[5], at::kFloat, at::IntArrayRef({tokens, top}), dout));
        uint8_t *const pd = address(dout), *const po = dy ? dy->at_() : nullptr;
        const int32_t *const pb = (const int32_t *)address(back);
        const float *const ps = (const float *)address(share);
        float *const pds = dshare ? (float *)dshare->at_() : nullptr;
        void *const s = stream();
        Py_BEGIN_ALLOW_THREADS
        gatherBackward(s, pd, py, pb, ps, po, pds, (uint32_t)tokens, (uint32_t)top, (uint32_t)cols, typeCode);
        Py_END_ALLOW_THREADS
        if (!accepted()) return nullptr;
        PyObject *const both = PyTuple_New(2);
        if (both == nullptr) return nullptr;
        std::optional<Result> *const made[2] = {&dy, &dshare};
        for (int i = 0; i < 2; ++i) {
            PyObject *o = *made[i] ? (**made[i]).object() : Py_None;
            if (!*made[i]) Py_INCREF(o);
            if (o == nullptr) {
                Py_DECREF(both);
                return nullptr;
            }
            PyTuple_SET_ITEM(both, i, o);
        }
        return both;
    });
}

PyMethodDef methods[] = {{"attach_ragged", (PyCFunction)(void *)attachRagged, METH_FASTCALL, "addresses of the e4m3 and grouped operators' functions"},
                         {"quantize_fp8", (PyCFunction)(void *)quantize, METH_FASTCALL, "one call: (codes, scale), or None for the Python path"},
                         {"fp8_matmul_allreduce", (PyCFunction)(void *)fp8, METH_FASTCALL, "one call: the output, or None for the Python path"},
                         {"grouped_matmul", (PyCFunction)(void *)grouped, METH_FASTCALL, "one call: the output, or None for the Python path"},
                         {"grouped_matmul_dw", (PyCFunction)(void *)dw, METH_FASTCALL, "one call: the output, or None for the Python path"},
                         {"grouped_fp8_matmul", (PyCFunction)(void *)fp8Grouped, METH_FASTCALL, "one call: the output, or None for the Python path"},
                         {"attach_layer", (PyCFunction)(void *)attachLayer, METH_FASTCALL, "addresses of the functions around a layer of experts"},
                         {"rms_norm", (PyCFunction)(void *)norm16, METH_FASTCALL, "one call: the output or outputs, or None for the Python path"},
                         {"rms_norm_fp8", (PyCFunction)(void *)normFp8, METH_FASTCALL, "one call: the outputs, or None for the Python path"},
                         {"rms_norm_backward", (PyCFunction)(void *)normBackward, METH_FASTCALL, "one call: (dx, dw), or None for the Python path"},
                         {"route", (PyCFunction)(void *)route, METH_FASTCALL, "one call: (choice, share), or None for the Python path"},
                         {"route_backward", (PyCFunction)(void *)routeGradient, METH_FASTCALL, "one call: the output, or None for the Python path"},
                         {"sort_by_expert", (PyCFunction)(void *)sortChoices, METH_FASTCALL, "one call: (order, back, ends), or None for the Python path"},
                         {"spread_rows", (PyCFunction)(void *)spread, METH_FASTCALL, "one call: the output or outputs, or None for the Python path"},
                         {"gather_rows", (PyCFunction)(void *)gather, METH_FASTCALL, "one call: the output, or None for the Python path"},
                         {"gather_rows_backward", (PyCFunction)(void *)gatherGradient, METH_FASTCALL, "one call: (dy, dshare), None for what is not wanted, or None for the Python path"},
                         {"attach", (PyCFunction)(void *)attach, METH_FASTCALL, "addresses of the library's functions, CatcocError, CocTilingParams"},
                         {"call", (PyCFunction)(void *)call, METH_FASTCALL, "one operator call: the output, or None for the Python path"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
