"""CPU suite: products in 8-bit integers and attention at the boundary, without a GPU: argument errors of the C entries and of the Python
mirror, how attention's work is shared out, the argument structures, and the operator list's new nodes."""
import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest
import torch

from dlf_b200 import gblas, gdnn, predict, tensor
from dlf_b200.gblas import BLASError, StatusCode

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p(0x1000)


def test_shares_of_attentions_work_and_argument_structures(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    exe = str(tmp_path / "plan")
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-o", exe, os.path.join(ROOT, "tests", "cpp", "test_attention_plan.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    sizes = [int(x) for x in out.stdout.split()]
    six, seven = gdnn._SIX_POINTERS.size, gdnn._SEVEN_POINTERS.size
    assert sizes == [gdnn._ATTENTION_ARGS.size, gdnn._ATTENTION_ARGS.size + six, gdnn._PAGED_ARGS.size, gdnn._PAGED_ARGS.size + six,
                     gdnn._APPEND_ARGS.size, gdnn._APPEND_ARGS.size + seven]


# ---------------------------------------------------------------------------------------------
# refusals of the C entries


def _quantize(L, dtype=16, m=4, n=8, x=P, x_ld=8, q=P, q_ld=8, s=P):
    return L.dlf_b200_quantize_rows(dtype, m, n, x, x_ld, q, q_ld, s, None)


def _product(L, dtype=32, m=4, n=4, k=16, a=P, a_ld=16, sa=P, b=P, b_ld=16, sb=P, act=0, c=P, c_ld=4, ws=None, nbytes=0):
    return L.dlf_b200_gemm_int8(dtype, m, n, k, a, a_ld, sa, b, b_ld, sb, None, act, c, c_ld, ws, nbytes, None)


def test_int8_argument_errors_without_a_device(built_lib):
    L = built_lib
    assert _quantize(L, dtype=64) == StatusCode.kNotImplemented
    assert _quantize(L, m=0) == StatusCode.kInvalidDimension
    assert _quantize(L, n=0) == StatusCode.kInvalidDimension
    assert _quantize(L, n=1 << 31, x_ld=1 << 31, q_ld=1 << 31) == StatusCode.kInvalidDimension
    assert _quantize(L, x_ld=7) == StatusCode.kInvalidLeadDimA
    assert _quantize(L, q_ld=7) == StatusCode.kInvalidLeadDimC
    assert _quantize(L, x=None) == StatusCode.kInvalidMatrixA
    assert _quantize(L, q=None) == _quantize(L, s=None) == StatusCode.kInvalidMatrixC
    assert _product(L, dtype=8) == StatusCode.kNotImplemented
    assert _product(L, act=2) == StatusCode.kInvalidValue
    assert _product(L, k=0) == StatusCode.kInvalidDimension
    assert _product(L, k=131072, a_ld=131072, b_ld=131072) == StatusCode.kInvalidDimension  # a sum could pass 32 bits
    assert _product(L, a_ld=15) == StatusCode.kInvalidLeadDimA
    assert _product(L, b_ld=15) == StatusCode.kInvalidLeadDimB
    assert _product(L, c_ld=3) == StatusCode.kInvalidLeadDimC
    assert _product(L, a=None) == _product(L, sa=None) == StatusCode.kInvalidMatrixA
    assert _product(L, b=None) == _product(L, sb=None) == StatusCode.kInvalidMatrixB
    assert _product(L, c=None) == StatusCode.kInvalidMatrixC
    # lines off 16-byte boundaries need room for their copies
    need = L.dlf_b200_gemm_int8_workspace_bytes(4, 4, 16, P, 17, P, 16)
    assert need >= 4 * 16 and L.dlf_b200_gemm_int8_workspace_bytes(4, 4, 16, P, 16, P, 32) == 0
    assert L.dlf_b200_gemm_int8_workspace_bytes(1, 1, 16, P, 17, P, 21) == 0  # one line each: only where it starts counts
    assert L.dlf_b200_gemm_int8_workspace_bytes(1, 1, 16, ctypes.c_void_p(0x1001), 16, P, 16) > 0
    assert _product(L, a_ld=17) == _product(L, a_ld=17, ws=P, nbytes=need - 1) == StatusCode.kInsufficientMemoryTemp


def _attention(L, dtype=16, scale=1.0, batch=2, queries=40, keys=6, heads=4, kv=2, size=64, strides=None, ptrs=None, mask=0, mask_ld=0, nbytes=1 << 30):
    st = strides or [queries * heads * size, heads * size, size] + 2 * [keys * kv * size, kv * size, size] + [queries * heads * size, heads * size, size]
    args = gdnn._ATTENTION_ARGS.pack(dtype, scale, batch, queries, keys, heads, kv, size, *st, mask_ld)
    p = list(ptrs or (0x1000,) * 4) + [0, mask]
    return L.dlf_b200_attention(args + gdnn._SIX_POINTERS.pack(*p), P if nbytes else None, nbytes, None)


def test_attention_argument_errors_without_a_device(built_lib):
    L = built_lib
    assert L.dlf_b200_attention(None, None, 0, None) == StatusCode.kInvalidValue
    for dtype in (32, 8):
        assert _attention(L, dtype=dtype) == StatusCode.kNotImplemented
    for size in (136, 12, 256):
        assert _attention(L, size=size) == StatusCode.kNotImplemented
    for kw in ({"batch": 0}, {"queries": 0}, {"keys": 0}, {"kv": 0}, {"kv": 3}, {"size": 0}, {"batch": 70000}):
        assert _attention(L, **kw) == StatusCode.kInvalidDimension, kw
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert _attention(L, scale=scale) == StatusCode.kInvalidValue
    for i, code in enumerate((StatusCode.kInvalidMatrixA, StatusCode.kInvalidMatrixB, StatusCode.kInvalidMatrixB, StatusCode.kInvalidMatrixC)):
        p = [0x1000] * 4
        p[i] = 0
        assert _attention(L, ptrs=p) == code
        p[i] = 0x1008  # off a 16-byte boundary
        assert _attention(L, ptrs=p) == StatusCode.kNotImplemented
    good = [10240, 256, 64] + 2 * [768, 128, 64] + [10240, 256, 64]
    for i in range(12):
        st = list(good)
        st[i] += 4
        assert _attention(L, strides=st) == StatusCode.kNotImplemented, i
        st[i] = 0
        code = {0: None, 3: None, 6: None}.get(i, (StatusCode.kInvalidLeadDimA, StatusCode.kInvalidLeadDimB, StatusCode.kInvalidLeadDimB, StatusCode.kInvalidLeadDimC)[i // 3])
        if code is not None:  # (a batch stride of 0 shares Q, K or V)
            assert _attention(L, strides=st) == code, i
    assert _attention(L, mask=0x1000, mask_ld=5) == StatusCode.kInvalidLeadDimB
    need = L.dlf_b200_attention_workspace_bytes(2, 1, 600, 4, 2, 64)
    assert need > 0 and _attention(L, queries=1, keys=600, nbytes=need - 1) == StatusCode.kInsufficientMemoryTemp
    assert L.dlf_b200_attention_workspace_bytes(2, 400, 128, 4, 2, 64) == 0  # one tile of keys: nothing is cut
    assert _attention(L, queries=400, keys=129, nbytes=0) == StatusCode.kInsufficientMemoryTemp


def _paged(L, dtype=16, scale=1.0, batch=2, heads=4, kv=2, size=64, pages=8, page=16, width=4, ld=4, st=None, ptrs=None, nbytes=1 << 30):
    st = st or [heads * size, size] + 2 * [page * kv * size, kv * size, size] + [heads * size, size]
    args = gdnn._PAGED_ARGS.pack(dtype, scale, batch, heads, kv, size, pages, page, width, ld, *st)
    return L.dlf_b200_paged_attention(args + gdnn._SIX_POINTERS.pack(*(ptrs or (0x1000,) * 6)), P if nbytes else None, nbytes, None)


def _append(L, dtype=16, tokens=2, kv=2, size=64, batch=2, pages=8, page=16, width=4, ld=4, st=None, ptrs=None):
    st = st or 2 * [kv * size, size] + 2 * [page * kv * size, kv * size, size]
    args = gdnn._APPEND_ARGS.pack(dtype, tokens, kv, size, batch, pages, page, width, ld, *st)
    return L.dlf_b200_paged_append(args + gdnn._SEVEN_POINTERS.pack(*(ptrs or (0x1000,) * 7)), None)


def test_paged_argument_errors_without_a_device(built_lib):
    L = built_lib
    assert L.dlf_b200_paged_attention(None, None, 0, None) == L.dlf_b200_paged_append(None, None) == StatusCode.kInvalidValue
    for f in (_paged, _append):
        assert f(L, dtype=32) == f(L, size=20) == f(L, size=136) == StatusCode.kNotImplemented
        for kw in ({"batch": 0}, {"kv": 0}, {"pages": 0}, {"page": 0}, {"width": 0}, {"size": 0}):
            assert f(L, **kw) == StatusCode.kInvalidDimension, kw
        assert f(L, ld=3) == StatusCode.kInvalidLeadDimB
    assert _paged(L, kv=3) == _paged(L, width=1 << 20, page=1 << 12, ld=1 << 20) == StatusCode.kInvalidDimension
    assert _paged(L, scale=-1.0) == StatusCode.kInvalidValue
    assert _append(L, tokens=0) == StatusCode.kInvalidDimension
    assert _append(L, tokens=3, ptrs=[0x1000] * 6 + [0]) == StatusCode.kInvalidDimension  # without sequences: one token for each
    for i, code in enumerate((StatusCode.kInvalidMatrixA, StatusCode.kInvalidMatrixB, StatusCode.kInvalidMatrixB, StatusCode.kInvalidMatrixC,
                              StatusCode.kInvalidMatrixB, StatusCode.kInvalidMatrixB)):
        p = [0x1000] * 6
        p[i] = 0
        assert _paged(L, ptrs=p) == code
    for i, code in enumerate((StatusCode.kInvalidMatrixA, StatusCode.kInvalidMatrixA, StatusCode.kInvalidMatrixC, StatusCode.kInvalidMatrixC,
                              StatusCode.kInvalidMatrixB, StatusCode.kInvalidMatrixB)):
        p = [0x1000] * 7
        p[i] = 0
        assert _append(L, ptrs=p) == code
        if i < 4:
            p[i] = 0x1004
            assert _append(L, ptrs=p) == StatusCode.kNotImplemented
    need = L.dlf_b200_paged_attention_workspace_bytes(2, 4, 2, 64)
    assert _paged(L, nbytes=need - 1) == StatusCode.kInsufficientMemoryTemp


# ---------------------------------------------------------------------------------------------
# refusals of the Python mirror


def _refused(code, f, *args, **kw):
    with pytest.raises(BLASError) as e:
        f(*args, **kw)
    assert e.value.status == code


def test_python_mirror_refuses_int8_calls_that_do_not_fit(built_lib):
    x, q, s = torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    with pytest.raises(tensor.ShapeError):
        tensor.quantize(x, q[:, :7], s)
    with pytest.raises(tensor.ShapeError):
        tensor.quantize(x, q, s[:3])
    with pytest.raises(tensor.ShapeError):
        tensor.quantize(x.t(), q.t().contiguous(), torch.zeros(8))
    _refused(StatusCode.kNotImplemented, tensor.quantize, x.double(), q, s)
    _refused(StatusCode.kInvalidMatrixA, tensor.quantize, x, q, s)  # not on a device
    _refused(StatusCode.kInvalidValue, gblas.quantizeRows, 4, 8, x, 0, 8, x, 0, 8, s)
    _refused(StatusCode.kInvalidDimension, gblas.quantizeRows, 0, 8, x, 0, 8, q, 0, 8, s)
    _refused(StatusCode.kInvalidLeadDimA, gblas.quantizeRows, 4, 8, x, 0, 7, q, 0, 8, s)
    _refused(StatusCode.kInsufficientMemoryA, gblas.quantizeRows, 4, 8, x, 1, 8, q, 0, 8, s)
    _refused(StatusCode.kInsufficientMemoryC, gblas.quantizeRows, 4, 8, x, 0, 8, q, 1, 8, s)
    _refused(StatusCode.kInsufficientMemoryC, gblas.quantizeRows, 4, 8, x, 0, 8, q, 0, 8, s[:3])
    a, sa, b, sb, c = q, s, torch.zeros(5, 8, dtype=torch.int8), torch.zeros(5), torch.zeros(4, 5)
    for bad in ((a[:, :7], sa, b, sb, c), (a, sa[:3], b, sb, c), (a, sa, b, sb[:4], c), (a, sa, b, sb, c[:3]), (a.t(), torch.zeros(8), b, sb, c)):
        with pytest.raises(tensor.ShapeError):
            tensor.matmul_int8(*bad)
    with pytest.raises(tensor.ShapeError):
        tensor.matmul_int8(a, sa, b, sb, c, bias=torch.zeros(4))
    _refused(StatusCode.kInvalidValue, tensor.matmul_int8, a, sa, b, sb, c, activation="gelu")
    _refused(StatusCode.kNotImplemented, tensor.matmul_int8, a, sa, b, sb, c.double())
    _refused(StatusCode.kInvalidMatrixA, tensor.matmul_int8, a, sa, b, sb, c)
    full = (4, 5, 8, a, 0, 8, sa, b, 0, 8, sb, c, 0, 5)
    for at, value, code in ((0, 0, StatusCode.kInvalidDimension), (5, 7, StatusCode.kInvalidLeadDimA), (9, 7, StatusCode.kInvalidLeadDimB),
                            (13, 4, StatusCode.kInvalidLeadDimC), (4, 1, StatusCode.kInsufficientMemoryA), (8, 1, StatusCode.kInsufficientMemoryB),
                            (12, 1, StatusCode.kInsufficientMemoryC), (6, sa[:3], StatusCode.kInsufficientMemoryA), (3, x, StatusCode.kInvalidValue)):
        args = list(full)
        args[at] = value
        _refused(code, gblas.gemmInt8, *args)


def test_python_mirror_refuses_attention_calls_that_do_not_fit(built_lib):
    def t(*shape, dtype=torch.float16):
        return torch.zeros(shape, dtype=dtype)

    q, k, y = t(2, 3, 4, 64), t(2, 6, 2, 64), t(2, 3, 4, 64)
    _refused(StatusCode.kInvalidMatrixA, gdnn.attention, q, k, k, y)  # not on a device
    with_shapes = [(t(2, 3, 4, 64, dtype=torch.bfloat16), k, k, y), (q, k, k.float(), y)]
    for bad in with_shapes:
        _refused(StatusCode.kInvalidValue, gdnn.attention, *bad)
    _refused(StatusCode.kInvalidDimension, gdnn.attention, q[0], k[0], k[0], y[0])
    pages, table, n = t(8, 16, 2, 64), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    _refused(StatusCode.kInvalidMatrixA, gdnn.paged_attention, q[:, 0], pages, pages, table, n, y[:, 0])
    _refused(StatusCode.kInvalidMatrixA, gdnn.paged_append, k[:, 0], k[:, 0], pages, pages, table, n)


# ---------------------------------------------------------------------------------------------
# the operator list


def test_attention_nodes_shapes():
    def shape(q, k, v=None, extra=(), **attrs):
        g = predict.Graph()
        node = g.append("Attention", **attrs)
        for name, d in (("q", q), ("k", k), ("v", v or k)):
            node.addInput(g.addInput(name, predict.DataType.FLOAT, d))
        for x in extra:
            node.addInput(None if x is None else g.addInput("n", predict.DataType.INT64, x))
        y = node.addOutput("y")
        predict.infer_shapes(g)
        assert not predict.unsupported_nodes(predict.optimize(g))
        return y.dims

    assert shape((2, 8, 5, 64), (2, 4, 9, 64)) == (2, 8, 5, 64)
    assert shape((2, 5, 512), (2, 9, 256), q_num_heads=8, kv_num_heads=4) == (2, 5, 512)
    assert shape((2, 8, 5, 64), (2, 4, 9, 64), extra=(None, None, None, (2,))) == (2, 8, 5, 64)
    for bad in (dict(q=(2, 8, 5, 64), k=(2, 3, 9, 64)), dict(q=(2, 8, 5, 64), k=(1, 8, 9, 64)), dict(q=(2, 8, 5, 64), k=(2, 8, 9, 32)),
                dict(q=(2, 5, 512), k=(2, 9, 512)), dict(q=(2, 8, 5, 64), k=(2, 8, 9, 64), v=(2, 8, 8, 64)),
                dict(q=(2, 8, 5, 64), k=(2, 8, 9, 64), is_causal=1), dict(q=(2, 8, 5, 64), k=(2, 8, 9, 64), extra=(None, None, None, (3,))),
                dict(q=(2, 8, 5, 64), k=(2, 8, 9, 64), extra=((2,),))):
        with pytest.raises(predict.ShapeInferenceError):
            shape(**bad)


def test_which_products_run_in_8_bit_integers():
    def graph(kind, a, w, c=None, c_known=True, relu=True, **attrs):
        g = predict.Graph()
        n = g.append(kind, **attrs)
        n.addInput(g.addInput("a", predict.DataType.FLOAT, a))
        n.addInput(g.addInitializer("w", np.zeros(w, np.float32)))
        if c is not None:
            n.addInput(g.addInitializer("c", np.zeros(c, np.float32)) if c_known else g.addInput("c", predict.DataType.FLOAT, c))
        y = n.addOutput("y")
        if relu:
            r = g.append("Relu")
            r.addInput(y)
            y = r.addOutput("r")
        g.addOutput(y)
        predict.infer_shapes(g)
        predict.optimize(g)
        return g

    for args in (("Gemm", (4, 8), (8, 6)), ("Gemm", (4, 8), (8, 6), (6,)), ("Gemm", (4, 8), (8, 6), (1, 6)), ("MatMul", (2, 4, 8), (8, 6))):
        g = graph(*args)
        assert predict.int8_product(g.nodes[0])
        assert predict.fuse_relu_into_int8_products(g)
        assert len(g.nodes) == 1 and g.nodes[0].attrs["relu"] and g.outputs[0] is g.nodes[0].output(0)
    for g in (graph("Gemm", (8, 4), (8, 6), transA=1), graph("Gemm", (4, 8), (8, 6), alpha=0.5), graph("Gemm", (4, 8), (8, 6), (4, 6)),
              graph("Gemm", (4, 8), (8, 6), (6,), c_known=False), graph("Gemm", (4, 8), (8, 6), (6,), beta=0.5), graph("MatMul", (2, 4, 8), (2, 8, 6)),
              graph("MatMul", (8,), (8, 6))):
        assert not predict.int8_product(g.nodes[0])
        assert not predict.fuse_relu_into_int8_products(g) and predict.unsupported_nodes(g)


def test_products_deeper_than_exact_sums_stay_in_floating_point():
    for k, exact in ((131071, True), (131072, False)):
        g = predict.Graph()
        n = g.append("MatMul")
        n.addInput(g.addInput("a", predict.DataType.FLOAT, (2, k)))
        n.addInput(g.addInitializer("w", np.zeros((k, 1), np.float32)))
        g.addOutput(n.addOutput("y"))
        predict.infer_shapes(g)
        assert predict.int8_product(g.nodes[0]) == exact


def test_attention_nodes_refuse_outputs_and_lengths_that_are_not_there():
    def graph():
        g = predict.Graph()
        node = g.append("Attention")
        for name in "qkv":
            node.addInput(g.addInput(name, predict.DataType.FLOAT, (2, 4, 5, 64)))
        node.addOutput("y")
        return g, node

    g, node = graph()
    node.addOutput("present_key")
    with pytest.raises(predict.ShapeInferenceError):
        predict.infer_shapes(g)
    g, node = graph()
    flat = predict.Node("Flatten", {"axis": 0})
    g.nodes.insert(0, flat)
    flat.addInput(g.addInput("n", predict.DataType.FLOAT, (2, 1)))
    for _ in range(3):
        node.addInput(None)
    node.addInput(flat.addOutput("lengths"))  # computed in floating point
    with pytest.raises(predict.ShapeInferenceError):
        predict.infer_shapes(g)


def test_integers_of_a_graph_keep_the_lists_type_unless_they_are_lengths():
    """Weights and inputs that are whole numbers are operands like others; lengths are 32-bit integers, cut to their range."""
    g = predict.Graph()
    n = g.append("MatMul")
    n.addInput(g.addInput("a", predict.DataType.INT64, (3, 4)))
    n.addInput(g.addInitializer("w", np.arange(8).reshape(4, 2)))
    g.addOutput(n.addOutput("p"))
    node = g.append("Attention")
    for name in "qkv":
        node.addInput(g.addInput(name, predict.DataType.FLOAT, (3, 2, 5, 64)))
    for _ in range(3):
        node.addInput(None)
    node.addInput(g.addInitializer("n", np.array([2 ** 32 + 5, -(2 ** 40), 4])))
    g.addOutput(node.addOutput("y"))
    p = predict.Predictor(g, torch.float16, device="cpu", cuda_graph=False)
    ops = {type(op).__name__: op for op in p.operators}
    assert ops["MatMulOp"].A.dtype == ops["MatMulOp"].B.dtype == torch.float16
    assert ops["MatMulOp"].B.tolist() == [[0, 1], [2, 3], [4, 5], [6, 7]]
    assert ops["AttentionOp"].lengths.dtype == torch.int32 and ops["AttentionOp"].lengths.tolist() == [2 ** 31 - 1, -1, 4]
    p.set(0, torch.arange(12).view(3, 4))
    assert p.input(0).tolist() == torch.arange(12).view(3, 4).tolist()


def test_lengths_that_are_set_are_cut_to_32_bits():
    g = predict.Graph()
    node = g.append("Attention")
    for name in "qkv":
        node.addInput(g.addInput(name, predict.DataType.FLOAT, (2, 2, 5, 64)))
    for _ in range(3):
        node.addInput(None)
    node.addInput(g.addInput("n", predict.DataType.INT64, (2,)))
    g.addOutput(node.addOutput("y"))
    p = predict.Predictor(g, torch.float16, device="cpu", cuda_graph=False)
    for given, want in ((torch.tensor([2 ** 32 + 3, -(2 ** 33)]), [2 ** 31 - 1, -1]), (torch.tensor([3, -1], dtype=torch.int8), [3, -1])):
        p.set(3, given)
        assert p.input(3).tolist() == want


def test_attention_scale_beyond_single_precision_is_refused(built_lib):
    assert _attention(built_lib, scale=3.0e38) == StatusCode.kInvalidValue  # (times log2 e)
    assert _paged(built_lib, scale=3.0e38) == StatusCode.kInvalidValue
    for scale in (3.0e38, 1e300):
        with pytest.raises(BLASError):
            gdnn._default_scale(scale, 64)


def test_a_scale_in_a_tensor_is_read_at_every_call(built_lib, monkeypatch):
    seen = []
    for plans in ("_ATTENTION_PLANS", "_PAGED_PLANS"):
        monkeypatch.setattr(gdnn, plans, gblas._Plans())
    monkeypatch.setattr(gdnn, "_placed", lambda *a: None)
    monkeypatch.setattr(gdnn, "_attention_call", lambda fn, args, *rest: seen.append(gdnn._ATTENTION_ARGS.unpack_from(args)[1]))
    q, scale = torch.zeros(1, 3, 2, 64, dtype=torch.float16), torch.tensor(0.5)
    for value in (0.5, 0.25):
        scale.fill_(value)
        gdnn.attention(q, q, q, torch.empty_like(q), scale=scale)
        gdnn.paged_attention(q[0], q, q, torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32), torch.empty_like(q[0]), scale=scale)
    assert seen == [0.5, 0.5, 0.25, 0.25]


def test_streams_of_another_device_are_refused():
    class Queue:
        device_index, cuda_stream = 1, 0

    _refused(StatusCode.kInvalidValue, gblas._operator_stream, Queue(), torch.device("cuda", 0))
    assert gblas._operator_stream(Queue(), torch.device("cuda", 1)) == 0


# ---------------------------------------------------------------------------------------------
# one graph, several lists


def _gemm_relu_graph():
    g = predict.Graph()
    n = g.append("Gemm")
    n.addInput(g.addInput("a", predict.DataType.FLOAT, (4, 8)))
    n.addInput(g.addInitializer("w", np.ones((8, 6), np.float32)))
    r = g.append("Relu")
    r.addInput(n.addOutput("y"))
    m = g.append("MatMul")
    m.addInput(r.addOutput("r"))
    m.addInput(g.addInitializer("w2", np.ones((6, 3), np.float32)))
    g.addOutput(m.addOutput("z"))
    return g


def _rounded_on_the_host(monkeypatch):
    """Lists of 8-bit products without a device: the weights are not rounded, only passed on."""
    monkeypatch.setattr(predict.linalg, "quantize", lambda W, *out: (W, torch.ones(W.shape[0])))


def test_a_list_of_8_bit_products_leaves_its_graph_as_it_was(monkeypatch):
    _rounded_on_the_host(monkeypatch)
    g = _gemm_relu_graph()
    for _ in range(2):
        with pytest.raises(NotImplementedError):  # a Relu behind a product in floating point is outside the library's path
            predict.Predictor(g, torch.float16, device="cpu", cuda_graph=False)
        p = predict.Predictor(g, torch.float16, device="cpu", cuda_graph=False, int8=True)
        assert [(type(op).__name__, op.relu) for op in p.operators] == [("Int8ProductOp", True), ("Int8ProductOp", False)]
        assert p.operators[0].Y is p.operators[1].A
        assert [n.kind for n in g.nodes] == ["Gemm", "Relu", "MatMul"] and not any(n.get("relu") for n in g.nodes)


def test_a_copied_graph_shares_nothing_that_a_pass_changes():
    g = predict.Graph()
    x, w = g.addInput("x", predict.DataType.FLOAT, (1, 8, 6, 6)), g.addInitializer("w", np.ones((8, 8, 1, 1), np.float32))
    values = [x]
    for name in ("a", "b"):
        n = g.append("Conv", kernel_shape=(1, 1))
        n.addInput(values[-1])
        n.addInput(w)
        values.append(n.addOutput(name))
    add = g.append("Add")
    add.addInput(values[2])
    add.addInput(values[1])
    g.addOutput(add.addOutput("y"))
    predict.infer_shapes(g)
    predict.optimize(g)
    assert g.nodes[1].attrs["residual"] is values[1]
    c = g.copy()
    assert c.inputs == g.inputs and c.inputs is not g.inputs
    a, b = c.nodes
    assert a.output(0) is not values[1] and a.output(0).dims == values[1].dims and a.output(0).node is a
    assert b.input(0) is a.output(0) and b.attrs["residual"] is a.output(0) and c.outputs == [b.output(0)]
    assert a.input(0) is x and a.input(1) is w
    assert [type(op).__name__ for op in predict.Predictor(c, torch.float32, device="cpu").operators] == ["ConvOp", "ConvOp"]


def test_a_graph_marked_for_8_bit_products_is_refused_in_floating_point(monkeypatch):
    _rounded_on_the_host(monkeypatch)
    g = predict.infer_shapes(_gemm_relu_graph())
    assert predict.fuse_relu_into_int8_products(g)
    with pytest.raises(NotImplementedError):
        predict.Predictor(g, torch.float16, device="cpu", cuda_graph=False)
    assert predict.Predictor(g, torch.float16, device="cpu", cuda_graph=False, int8=True).operators[0].relu


@pytest.mark.parametrize("name", ["attention_decode.cuh", "attention_short.cuh", "attention_tiles.cuh", "contraction_int8.cuh", "quantize.cuh"])
def test_kernels_read_no_device_memory_before_they_wait_for_the_kernel_before_them(name):
    """A programmatic dependent may start while the kernel before it runs: what others wrote is visible behind the wait only."""
    with open(os.path.join(ROOT, "dlf_b200", "csrc", name)) as f:
        kernels = re.findall(r"__global__.*?\n}\n", f.read(), re.S)
    assert kernels
    for body in kernels:
        before, wait, _ = body.partition("wait_for_dependencies();")
        assert wait, body[:200]
        assert not re.search(r"plan_(sums|find|sequence)\(|PlanWalk walk|p\.(lengths|table|positions|sequences|mask|sa|sb)\[|\*reinterpret_cast<const", before), before[-400:]


def test_workspaces_have_room_for_a_start_anywhere(built_lib):
    """The parts of cut sequences (16 or 256 rows of size + 2 floats, two for each CTA) start on 16 bytes wherever the workspace does."""
    L = built_lib
    for size, ctas in ((8, 592), (64, 592), (72, 444), (128, 444)):
        parts = ctas * (2 * 16 * (size + 2) * 4 + 16)
        assert L.dlf_b200_paged_attention_workspace_bytes(3, 4, 2, size) >= parts + 15
        assert L.dlf_b200_attention_workspace_bytes(3, 1, 600, 4, 2, size) >= parts + 15
        assert L.dlf_b200_attention_workspace_bytes(3, 500, 600, 4, 2, size) >= 2 * 148 * 256 * (size + 2) * 4 + 15


def test_a_list_of_8_bit_products_keeps_no_other_weights(monkeypatch):
    """But for those that an operator in floating point reads as well."""
    _rounded_on_the_host(monkeypatch)
    g = _gemm_relu_graph()
    shared = g.addInitializer("w3", np.ones((3, 3), np.float32))
    m = g.append("MatMul")
    m.addInput(g.outputs.pop())
    m.addInput(shared)
    z = m.addOutput("u")
    n = g.append("MatMul")  # weights times a value: in floating point
    n.addInput(shared)
    n.addInput(g.addInput("b", predict.DataType.FLOAT, (3, 2)))
    for v in (z, n.addOutput("v")):
        g.addOutput(v)
    p = predict.Predictor(g, torch.float16, device="cpu", cuda_graph=False, int8=True)
    assert [type(op).__name__ for op in p.operators] == ["Int8ProductOp"] * 3 + ["MatMulOp"]
    weights = {id(v): v.name for v in g.inputs if v.has_initializer()}
    assert [weights[i] for i in p._data if i in weights] == ["w3"]


def test_results_allocated_for_another_stream_come_from_its_memory(built_lib, monkeypatch):
    entered, allocated = [], []

    class Stream:
        def __init__(self, queue):
            self.queue = queue

        def __enter__(self):
            entered.append(self.queue)

        def __exit__(self, *exc):
            entered.pop()

    class Queue:
        device_index, cuda_stream = 0, 0

    empty, queue = torch.empty, Queue()
    monkeypatch.setattr(torch.cuda, "stream", Stream)
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: (allocated.append(list(entered)), empty(*a, **kw))[1])
    x, q, s = torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    for given, want in ((queue, [queue]), (None, [])):
        allocated.clear()
        _refused(StatusCode.kInvalidMatrixA, tensor.quantize, x, queue=given)  # (not on a device)
        _refused(StatusCode.kInvalidMatrixA, tensor.matmul_int8, q, s, q, s, queue=given)
        assert allocated == [want] * 3


def test_a_streams_scratch_comes_from_its_memory(monkeypatch):
    entered, allocated, queue = [], [], object()

    class Stream:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            entered.append(self.stream)

        def __exit__(self, *exc):
            entered.pop()

    empty = torch.empty
    monkeypatch.setattr(torch.cuda, "stream", Stream)
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: (allocated.append(list(entered)), empty(*a, **kw))[1])
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, stream: None)
    scratch = gblas._StreamScratch()
    for nbytes in (100, 50, 200):
        assert scratch.at_least(nbytes, torch.device("cpu"), queue).numel() >= nbytes
    assert allocated == [[queue]] * 2


def test_other_calls_on_another_stream_take_that_streams_memory(monkeypatch):
    """Packed filters, channels-last copies, the tables and the scratch of batched products and of level 3."""
    entered, allocated = [], []

    class Stream:
        def __init__(self, queue):
            self.queue = queue

        def __enter__(self):
            entered.append(self.queue)

        def __exit__(self, *exc):
            entered.pop()

    class Queue:
        device_index, cuda_stream = 0, 0

    class Library:
        def __getattr__(self, name):
            return lambda *args: 64 if name.endswith(("_bytes", "_elems")) else 0

    empty, queue = torch.empty, Queue()
    monkeypatch.setattr(torch.cuda, "stream", Stream)
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: (allocated.append(list(entered)), empty(*a, **kw))[1])
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, stream: None)
    for module in (gblas, gdnn):
        monkeypatch.setattr(module, "lib", Library)
        monkeypatch.setattr(module, "_ptr", lambda buf, offset=0: buf.data_ptr())
    x = torch.zeros(1, 8, 4, 4)
    gdnn.pack_filters_nhwc(x, queue=queue)
    gdnn.nchw_to_nhwc(x, queue=queue)
    m = torch.zeros(16)
    gblas.gemmBatched(gblas.Layout.RowMajor, gblas.Transpose.NoTrans, gblas.Transpose.NoTrans, 4, 4, 4, [1.0], m, [0], 4, m, [0], 4, [0.0], m, [0], 4, 1,
                      queue=queue)
    gblas.symm(gblas.Layout.RowMajor, gblas.Side.Left, gblas.Triangle.Upper, 4, 4, 1.0, m, 0, 4, m, 0, 4, 0.0, m, 0, 4, queue=queue)
    assert allocated == [[queue]] * 4
