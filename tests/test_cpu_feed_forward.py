"""Gated and 8-bit products without a GPU: shape rules and refusals, fusion,
candidates."""

from __future__ import annotations

import numpy as np
import pytest

import cutriton_b200 as ct
import feed_forward_cases as ff


@pytest.fixture(autouse=True)
def assume_sm100(monkeypatch):
    monkeypatch.setenv("CUTRITON_ASSUME_COMPUTE_CAPABILITY", "100")


def zeros(**shapes):
    """name=(dtype, shape) -> arrays, in order."""
    return {name: np.zeros(shape, dtype) for name, (dtype, shape) in shapes.items()}


GATED = dict(x=("f2", (4, 32)), w_gate=("f2", (24, 32)), w_up=("f2", (24, 32)))
QGEMM = dict(x=("i1", (4, 32)), x_scale=("f4", (4,)), w=("i1", (24, 32)), w_scale=("f4", (24,)))
QGATED = dict(x=("i1", (4, 32)), x_scale=("f4", (4,)), w_gate=("i1", (24, 32)), gate_scale=("f4", (24,)),
              w_up=("i1", (24, 32)), up_scale=("f4", (24,)))


@pytest.mark.parametrize("op,inputs", [("GatedGemm", GATED), ("QGemm", QGEMM), ("QGatedGemm", QGATED),
                                       ("QGemm", {**QGEMM, "bias": ("f2", (24,))})])
def test_outputs_are_described(op, inputs):
    engine = ct.build_engine(ff.product_graph(op, zeros(**inputs), transB=1))
    assert engine.value_desc("y") == (ct.FLOAT16, (4, 24))
    turned = {n: (d, s[::-1] if n.startswith("w") and len(s) == 2 else s) for n, (d, s) in inputs.items()}
    engine = ct.build_engine(ff.product_graph(op, zeros(**turned), transB=0))
    assert engine.value_desc("y") == (ct.FLOAT16, (4, 24))


def test_quantize_rows_has_two_outputs():
    engine = ct.build_engine(ff.product_graph("QuantizeRows", zeros(x=("f2", (4, 33)))))
    assert engine.value_desc("q") == (ct.INT8, (4, 33))
    assert engine.value_desc("q_scale") == (ct.FLOAT32, (4,))


@pytest.mark.parametrize("op,inputs,attributes,code", [
    ("GatedGemm", {**GATED, "w_up": ("f2", (25, 32))}, {}, ct.SHAPE_ERROR),
    ("GatedGemm", {**GATED, "w_gate": ("f2", (24, 31))}, {}, ct.SHAPE_ERROR),
    ("GatedGemm", {**GATED, "w_gate": ("f2", (24, 32, 1))}, {}, ct.SHAPE_ERROR),
    ("GatedGemm", {**GATED, "w_gate": ("f4", (24, 32))}, {}, ct.SHAPE_ERROR),
    ("GatedGemm", {**GATED, "x": ("f2", (2, 2, 32))}, {}, ct.SHAPE_ERROR),
    ("GatedGemm", {n: ("f4", s) for n, (_, s) in GATED.items()}, {}, ct.UNSUPPORTED),
    ("GatedGemm", {n: ("i1", s) for n, (_, s) in GATED.items()}, {}, ct.UNSUPPORTED),
    ("GatedGemm", GATED, {"activation": 2}, ct.UNSUPPORTED),
    ("GatedGemm", GATED, {"activation": -1}, ct.UNSUPPORTED),
    ("GatedGemm", GATED, {"transB": 2}, ct.UNSUPPORTED),
    ("GatedGemm", GATED, {"transA": 1}, ct.UNSUPPORTED),
    ("QGemm", {**QGEMM, "x": ("f2", (4, 32))}, {}, ct.SHAPE_ERROR),
    ("QGemm", {**QGEMM, "w": ("f2", (24, 32))}, {}, ct.SHAPE_ERROR),
    ("QGemm", {**QGEMM, "w": ("i1", (24, 48))}, {}, ct.SHAPE_ERROR),
    ("QGemm", {**QGEMM, "x_scale": ("f4", (5,))}, {}, ct.SHAPE_ERROR),
    ("QGemm", {**QGEMM, "x_scale": ("f4", (4, 1))}, {}, ct.SHAPE_ERROR),
    ("QGemm", {**QGEMM, "w_scale": ("f2", (24,))}, {}, ct.SHAPE_ERROR),
    ("QGemm", {**QGEMM, "w_scale": ("f4", (32,))}, {}, ct.SHAPE_ERROR),
    ("QGemm", {**QGEMM, "bias": ("f4", (24,))}, {}, ct.SHAPE_ERROR),
    ("QGemm", {**QGEMM, "bias": ("f2", (4, 24))}, {}, ct.SHAPE_ERROR),
    ("QGemm", {**QGEMM, "x": ("i1", (4, 131072)), "w": ("i1", (24, 131072))}, {}, ct.UNSUPPORTED),
    ("QGatedGemm", {**QGATED, "up_scale": ("f4", (23,))}, {}, ct.SHAPE_ERROR),
    ("QGatedGemm", {**QGATED, "w_up": ("i1", (23, 32)), "up_scale": ("f4", (23,))}, {}, ct.SHAPE_ERROR),
    ("QGatedGemm", QGATED, {"activation": 3}, ct.UNSUPPORTED),
    ("QuantizeRows", {"x": ("f4", (4, 32))}, {}, ct.SHAPE_ERROR),
    ("QuantizeRows", {"x": ("f2", (4, 32, 2))}, {}, ct.SHAPE_ERROR),
    ("QuantizeRows", {"x": ("i1", (4, 32))}, {}, ct.SHAPE_ERROR),
])
def test_refusals(op, inputs, attributes, code):
    attributes = {"transB": 1, **attributes} if op != "QuantizeRows" else attributes
    with pytest.raises(ct.CutritonError) as error:
        ct.build_engine(ff.product_graph(op, zeros(**inputs), **attributes))
    assert error.value.code == code, error.value


@pytest.mark.parametrize("op,inputs", [("QGemm", {n: QGEMM[n] for n in ("x", "x_scale", "w")}),
                                       ("QGatedGemm", {n: QGATED[n] for n in list(QGATED)[:5]}),
                                       ("GatedGemm", {n: GATED[n] for n in ("x", "w_gate")})])
def test_missing_inputs_are_refused(op, inputs):
    with pytest.raises(ct.CutritonError) as error:
        ct.build_engine(ff.product_graph(op, zeros(**inputs), transB=1))
    assert error.value.code == ct.SHAPE_ERROR


@pytest.mark.parametrize("op", ["Relu", "Add", "Gemm", "Softmax", "GlobalAveragePool"])
def test_other_ops_take_no_int8(op):
    model = ct.Model()
    shape = [1, 4, 4, 4] if op == "GlobalAveragePool" else [4, 4]
    names = ["a", "b"] if op in ("Add", "Gemm") else ["a"]
    for name in names:
        model.add_input(name, shape, dtype=np.int8, layout="NCHW" if len(shape) == 4 else "")
    model.add_node("node", op, names, ["y"])
    model.add_output("y")
    with pytest.raises(ct.CutritonError) as error:
        ct.build_engine(model)
    assert error.value.code == ct.UNSUPPORTED


def gated_chain(activation="Silu", swap=False, extra_output=None, dtype=np.float16, other_input=False, reuse=False):
    model = ct.Model()
    model.add_input("x", [6, 32], dtype=dtype, layout="")
    model.add_input("z", [6, 32], dtype=dtype, layout="")
    for name in ("w_gate", "w_up"):
        model.add_constant(name, np.zeros((32, 24), dtype), layout="")
    model.add_node("gate", "MatMul" if swap else "Gemm", ["x", "w_gate"], ["g"])
    model.add_node("act", activation, ["g"], ["a"])
    model.add_node("up", "Gemm", ["z" if other_input else "x", "w_up"], ["u"])
    model.add_node("product", "Mul", ["u", "a"] if swap else ["a", "u"], ["y"])
    if reuse:
        model.add_node("again", "Add", ["u", "y"], ["sum"])
        model.add_output("sum")
    model.add_output("y")
    if extra_output:
        model.add_output(extra_output)
    return model


@pytest.mark.parametrize("activation,swap", [("Silu", False), ("Gelu", False), ("Silu", True), ("Gelu", True)])
def test_gated_chain_becomes_one_op(activation, swap):
    engine = ct.build_engine(gated_chain(activation, swap))
    (op,) = engine.ops()
    assert op["op_type"] == "GatedGemm" and op["node"] == "gate_gated"
    assert "unfused:gated_gemm" in op["candidates"]
    assert not op["candidates"][op["default"]].startswith("unfused")


@pytest.mark.parametrize("kwargs", [dict(extra_output="g"), dict(extra_output="u"), dict(extra_output="a"),
                                    dict(other_input=True), dict(reuse=True)])
def test_chain_whose_values_are_used_elsewhere_stays(kwargs):
    engine = ct.build_engine(gated_chain(**kwargs))
    assert "GatedGemm" not in [op["op_type"] for op in engine.ops()]


def test_transformer_fusions_off_keeps_the_chain():
    engine = ct.build_engine(gated_chain(), enable_transformer_fusions=0)
    assert [op["op_type"] for op in engine.ops()] == ["Gemm", "Silu", "Gemm", "Mul"]


def test_square_of_one_projection_is_not_a_gated_pair():
    model = ct.Model()
    model.add_input("x", [6, 32], dtype=np.float16, layout="")
    model.add_constant("w", np.zeros((32, 24), np.float16), layout="")
    model.add_node("gate", "Gemm", ["x", "w"], ["g"])
    model.add_node("act", "Silu", ["g"], ["a"])
    model.add_node("product", "Mul", ["a", "g"], ["y"])
    model.add_output("y")
    assert [op["op_type"] for op in ct.build_engine(model).ops()] == ["Gemm", "Silu", "Mul"]
