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


HUGE = 2**31 - 1024


@pytest.mark.parametrize("op,shapes", [
    ("GatedGemm", dict(x=("f2", (HUGE, 8)), w_gate=("f2", (24, 8)), w_up=("f2", (24, 8)))),
    ("GatedGemm", dict(x=("f2", (4, 8)), w_gate=("f2", (HUGE, 8)), w_up=("f2", (HUGE, 8)))),
    ("GatedGemm", dict(x=("f2", (4, HUGE)), w_gate=("f2", (24, HUGE)), w_up=("f2", (24, HUGE)))),
    ("QGemm", dict(x=("i1", (HUGE, 8)), x_scale=("f4", (HUGE,)), w=("i1", (24, 8)), w_scale=("f4", (24,)))),
    ("QGemm", dict(x=("i1", (4, 8)), x_scale=("f4", (4,)), w=("i1", (HUGE, 8)), w_scale=("f4", (HUGE,)))),
    ("QuantizeRows", dict(x=("f2", (HUGE, 2)))),
    ("QuantizeRows", dict(x=("f2", (2, HUGE)))),
])
def test_dimensions_whose_last_tile_passes_32_bits_are_refused(op, shapes):
    def build(shapes):
        model = ct.Model()
        for name, (dtype, shape) in shapes.items():
            model.add_input(name, list(shape), dtype=dtype, layout="")
        outs = ["q", "s"] if op == "QuantizeRows" else ["y"]
        model.add_node("node", op, list(shapes), outs, **({} if op == "QuantizeRows" else {"transB": 1}))
        for name in outs:
            model.add_output(name)
        return ct.build_engine(model)

    with pytest.raises(ct.CutritonError) as error:
        build(shapes)
    assert error.value.code == ct.UNSUPPORTED and "2^31 - 1024" in str(error.value)
    build({n: (d, tuple(v - 1 if v == HUGE else v for v in s)) for n, (d, s) in shapes.items()})


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


@pytest.mark.parametrize("trans_b,fused", [(0, False), (1, True)])
def test_weights_that_are_graph_inputs_fuse_by_rows_only(trans_b, fused):
    model = ct.Model()
    model.add_input("x", [6, 32], dtype=np.float16, layout="")
    for name in ("wg", "wu"):
        model.add_input(name, [24, 32] if trans_b else [32, 24], dtype=np.float16, layout="")
    model.add_node("gate", "Gemm", ["x", "wg"], ["g"], transB=trans_b)
    model.add_node("act", "Silu", ["g"], ["a"])
    model.add_node("up", "Gemm", ["x", "wu"], ["u"], transB=trans_b)
    model.add_node("product", "Mul", ["a", "u"], ["y"])
    model.add_output("y")
    ops = [o["op_type"] for o in ct.build_engine(model).ops()]
    assert ops == (["GatedGemm"] if fused else ["Gemm", "Silu", "Gemm", "Mul"])


def test_unfused_candidate_needs_two_buffers():
    """Gate and up projection share a slot: 2 x 6 x 24 FP16 in 256-byte slots."""
    assert ct.build_engine(gated_chain()).workspace_bytes() == 2 * 512


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


def test_few_row_form_is_a_candidate_of_every_plan():
    """Its row limit holds or not at a run's shapes, so lowering admits it and
    keeps the default; unfused steps never use it."""
    engine = ct.build_engine(ff.product_graph("QGemm", zeros(**QGEMM), transB=1))
    (op,) = engine.ops()
    assert any(".stream:" in c for c in op["candidates"])
    assert ".pair:" in op["candidates"][op["default"]]


@pytest.mark.parametrize("k", [31, 17])
def test_inner_sizes_off_16_bytes_take_the_general_form(k):
    shapes = {n: (d, tuple(k if e == 32 else e for e in s)) for n, (d, s) in QGEMM.items()}
    (op,) = ct.build_engine(ff.product_graph("QGemm", zeros(**shapes), transB=1)).ops()
    assert len(op["candidates"]) == 1 and ".any:" in op["candidates"][0]


@pytest.mark.parametrize("n,split", [(1, 8), (1536, 8), (1537, 4), (9472, 4), (9473, 2), (18944, 2), (18945, 1)])
def test_one_split_of_k_for_each_width(n, split):
    shapes = dict(x=("f2", (20, 32)), w_gate=("f2", (n, 32)), w_up=("f2", (n, 32)))
    engine = ct.build_engine(ff.product_graph("GatedGemm", zeros(**shapes), transB=1))
    narrow = [c for c in engine.op(0)["candidates"] if ".narrow" in c]
    assert len(narrow) == 1 and f".narrow{split}:" in narrow[0]


def test_at_run_constraint_is_part_of_the_pack_schema():
    from cutriton_b200 import kernel_sdk, kernel_specs

    specs = [s for s in kernel_specs.all_specs() if s.kernel_id.endswith(".stream")]
    assert len(specs) == 3
    for spec in specs:
        assert any(c.get("at_run") == 1 and c["value"] == 16 for c in spec.constraints)
        kernel_sdk.KernelSpec.validate(spec)


def test_launch_shapes_match_the_kernels():
    """Block sizes, shared memory and boxes that the pack gives and the kernels
    were compiled for."""
    import re
    from pathlib import Path

    from cutriton_b200 import kernel_specs

    folder = Path(kernel_specs.__file__).resolve().parent / "csrc" / "kernels"

    def constant(source, name):
        return int(re.search(rf"constexpr (?:int|uint32_t) {name} = (\d+);", (folder / source).read_text()).group(1))

    for spec in kernel_specs.all_specs():
        for variant in spec.variants:
            if spec.source == "product_pair.cu":
                assert variant.num_warps == 2 + constant(spec.source, "kEpilogueWarps")
                boxes = {a.name: a.source["box"] for a in spec.arguments if a.source["kind"] == "tensor_map"}
                block = 64 if ".fp16." in spec.kernel_id else 128
                assert [boxes[f"tma_x{r}"] for r in (128, 64, 32)] == [[block, r] for r in (128, 64, 32)]
                for name in ("w",) if spec.op_type == "QGemm" else ("gate", "up"):
                    assert [boxes[f"tma_{name}{r}"] for r in (128, 96, 64, 48, 32)] == \
                        [[block, r] for r in (128, 96, 64, 48, 32)]
                need = constant(spec.source, "kRingBytes") + 16 * 32 * 32 * 2 + 200 + 1024
                assert need <= variant.shared_memory_bytes <= 232448
            elif spec.source == "product_stream.cu":
                readers = 16 if spec.op_type == "QGemm" else 12
                name = "kPlainThreads" if spec.op_type == "QGemm" else "kGatedThreads"
                assert f"constexpr int {name} = ({readers} + kJoinWarps) * 32;" in (folder / spec.source).read_text()
                assert variant.num_warps == readers + constant(spec.source, "kJoinWarps")
                assert variant.shared_memory_bytes == constant(spec.source, "kSharedBytes") <= 232448
            elif spec.source == "product_narrow.cu":
                assert variant.num_warps * 32 == constant(spec.source, "kThreads")
                assert variant.shared_memory_bytes >= constant(spec.source, "kRingBytes") + 100 + 1023
                assert 2 * (variant.shared_memory_bytes + 1024) <= 228 * 1024  # two blocks an SM
                boxes = {a.name: a.source["box"][1] for a in spec.arguments if a.source["kind"] == "tensor_map"}
                assert boxes.pop("tma_x64") == 64 and boxes.pop("tma_x32") == 32 and set(boxes.values()) == {128}
            elif spec.source == "quantize.cu":
                warps = constant(spec.source, "kWarps")
                assert variant.num_warps == warps
                assert variant.shared_memory_bytes >= warps * (constant(spec.source, "kSlots") * 512 + 4)


def test_workload_blocks_lower_to_the_operators():
    from cutriton_b200 import workloads

    weights = workloads.gated_ffn_weights(64, 160)
    assert [o["op_type"] for o in ct.build_engine(workloads.build_gated_ffn(weights, 5)).ops()] == \
        ["GatedGemm", "Gemm", "SkipLayerNormalization"]
    assert [o["op_type"] for o in ct.build_engine(workloads.build_gated_ffn_int8(weights, 5)).ops()] == \
        ["QuantizeRows", "QGatedGemm", "QuantizeRows", "QGemm", "SkipLayerNormalization"]


def test_quantized_weight_holds_its_values():
    from cutriton_b200 import workloads

    weight = workloads.gated_ffn_weights(48, 40)["w_gate"]
    weight[:, 7] = 0
    rows, scale = workloads.quantize_weight(weight)
    assert rows.dtype == np.int8 and rows.shape == (40, 48) and scale[7] == 0 and not rows[7].any()
    # Half a step of the channel's scale (and the scale's own rounding).
    error = np.abs(rows * scale.astype(np.float64)[:, None] - weight.T.astype(np.float64))
    assert (error <= scale[:, None] * (0.5 + 128 * 2.0**-24)).all()


@pytest.mark.parametrize("activation", ["silu", "gelu", 0, 1], ids=str)
def test_facade_takes_the_operators(tmp_path, activation):
    import json

    from cutriton_b200 import api

    graph = {"inputs": ["x"], "outputs": ["y"], "input_shapes": {"x": [-1, 16]}, "input_dtypes": {"x": "float16"},
             "nodes": [{"name": "q", "op_type": "QuantizeRows", "inputs": ["x"], "outputs": ["x8", "xs"]},
                       {"name": "g", "op_type": "QGatedGemm", "inputs": ["x8", "xs", "wg", "gs", "wu", "us"],
                        "outputs": ["y"], "activation": activation, "transB": 1}],
             "constants": {**{n: {"data": [1] * 128, "shape": [8, 16], "dtype": "int8"} for n in ("wg", "wu")},
                           **{n: {"data": [0.5] * 8, "shape": [8], "dtype": "float32"} for n in ("gs", "us")}}}
    path = tmp_path / "g.json"
    path.write_text(json.dumps(graph))
    native = api.compile(path).native({"x": (3, 16)})
    assert [o["op_type"] for o in native.ops()] == ["QuantizeRows", "QGatedGemm"]
    assert native.value_desc("y") == (ct.FLOAT16, (3, 8))


def test_facade_refuses_other_activations(tmp_path):
    import json

    from cutriton_b200 import api

    graph = {"inputs": ["x", "a", "b"], "outputs": ["y"], "input_dtypes": {n: "float16" for n in "xab"},
             "nodes": [{"name": "g", "op_type": "GatedGemm", "inputs": ["x", "a", "b"], "outputs": ["y"],
                        "activation": None}]}
    path = tmp_path / "g.json"
    for activation in ("tanh", 2, [0]):
        graph["nodes"][0]["activation"] = activation
        path.write_text(json.dumps(graph))
        with pytest.raises(api.UnsupportedModelError):
            api.compile(path).native({"x": (3, 16), "a": (16, 8), "b": (16, 8)})


def test_scale_without_a_reader_is_planned():
    model = ct.Model()
    model.add_input("x", [4, 32], dtype=np.float16, layout="")
    model.add_node("quantize", "QuantizeRows", ["x"], ["q", "unused"])
    model.add_output("q")
    engine = ct.build_engine(model)
    assert engine.workspace_bytes() >= 16


def test_quantize_rows_needs_both_outputs():
    model = ct.Model()
    model.add_input("x", [4, 32], dtype=np.float16, layout="")
    model.add_node("quantize", "QuantizeRows", ["x"], ["q"])
    model.add_output("q")
    with pytest.raises(ct.CutritonError) as error:
        ct.build_engine(model)
    assert error.value.code == ct.SHAPE_ERROR


def test_one_matrix_may_be_both_weights():
    model = ct.Model()
    model.add_input("x", [4, 32], dtype=np.float16, layout="")
    model.add_constant("w", np.zeros((24, 32), np.float16), layout="")
    model.add_node("node", "GatedGemm", ["x", "w", "w"], ["y"], transB=1)
    model.add_output("y")
    assert ct.build_engine(model).value_desc("y") == (ct.FLOAT16, (4, 24))


def test_kernels_that_start_early_read_no_tensor_as_constant():
    """Under programmatic launch a grid starts while the kernel in front of it
    still writes, so its tensors are not constant while it runs: no
    read-only-path loads in the sources of the forms that ask for it."""
    from pathlib import Path

    from cutriton_b200 import kernel_specs

    folder = Path(kernel_specs.__file__).resolve().parent / "csrc" / "kernels"
    ops = ("GatedGemm", "QGemm", "QGatedGemm", "QuantizeRows")
    sources = {s.source for s in kernel_specs.all_specs() if s.op_type in ops and any(v.programmatic_launch for v in s.variants)}
    assert sources == {"product_pair.cu", "product_stream.cu", "product_narrow.cu", "quantize.cu"}
    for name in sources | {"product.cuh"}:
        text = (folder / name).read_text()
        assert "__ldg" not in text and "__restrict__" not in text and "ld.global.nc" not in text, name


@pytest.mark.parametrize("op", ["GatedGemm", "QGemm", "QGatedGemm"])
@pytest.mark.parametrize("attribute", [{"transA": 1}, {"alpha": 0.5}], ids=str)
def test_facade_refuses_a_turned_or_scaled_left_operand(tmp_path, op, attribute):
    """Square operands, whose shapes fit either way round."""
    import json

    from cutriton_b200 import api

    half = op == "GatedGemm"
    names = {"GatedGemm": ["x", "a", "b"], "QGemm": ["x", "s", "a", "t"], "QGatedGemm": ["x", "s", "a", "t", "b", "t"]}[op]
    dtypes = {n: "float32" if n in "st" else "float16" if half else "int8" for n in names}
    graph = {"inputs": sorted(set(names)), "outputs": ["y"], "input_dtypes": dtypes,
             "nodes": [{"name": "g", "op_type": op, "inputs": names, "outputs": ["y"]}]}
    shapes = {n: (16,) if n in "st" else (16, 16) for n in names}
    path = tmp_path / "g.json"
    path.write_text(json.dumps(graph))
    assert api.compile(path).native(shapes).value_desc("y") == (ct.FLOAT16, (16, 16))
    graph["nodes"][0].update(attribute)
    path.write_text(json.dumps(graph))
    with pytest.raises(api.UnsupportedModelError):
        api.compile(path).native(shapes)


def test_narrow_variants_are_named_by_the_rows_they_take():
    from cutriton_b200 import kernel_specs

    for spec in kernel_specs.all_specs():
        if spec.source == "product_narrow.cu":
            (most,) = [c["value"] for c in spec.constraints if c["kind"] == "dim_le" and c["source"] == "input"]
            assert [v.variant_id for v in spec.variants] == [f"rows{most}", f"rows{most}_turned"], spec.kernel_id
