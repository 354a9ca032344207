"""Graphs, inputs and 64-bit results of the gated and 8-bit products, with
the tolerances their FP32 arithmetic and one FP16 rounding allow."""

from __future__ import annotations

import numpy as np

import cutriton_b200 as ct

HALF = 2.0**-11  # FP16: half a step relative to the value
HALF_MIN = 2.0**-25  # half the smallest FP16 step

SILU, GELU = 0, 1


def erf64(x: np.ndarray) -> np.ndarray:
    import torch

    return torch.erf(torch.from_numpy(np.ascontiguousarray(x))).numpy()


def activate(g: np.ndarray, activation: int) -> np.ndarray:
    if activation == SILU:
        return g * 0.5 * (1.0 + np.tanh(g / 2))
    return 0.5 * g * (1.0 + erf64(g / np.sqrt(2.0)))


def product_graph(op: str, inputs: dict[str, np.ndarray], constants: tuple[str, ...] = (), **attributes) -> ct.Model:
    """One node `op` over `inputs` (in the node's order); those named in
    `constants` are model constants, the others graph inputs."""
    model = ct.Model()
    for name, array in inputs.items():
        if name in constants:
            model.add_constant(name, array, layout="")
        else:
            model.add_input(name, list(array.shape), dtype=array.dtype, layout="")
    outputs = ["q", "q_scale"] if op == "QuantizeRows" else ["y"]
    model.add_node("node", op, list(inputs), outputs, **attributes)
    for name in outputs:
        model.add_output(name)
    return model


def quantized(rng: np.random.Generator, rows: int, k: int) -> tuple[np.ndarray, np.ndarray]:
    """8-bit rows over the whole range, -128 included, and positive scales."""
    return (rng.integers(-128, 128, (rows, k)).astype(np.int8),
            (rng.uniform(0.5, 1.5, rows) * 0.3 / np.sqrt(k) / 40).astype(np.float32))


def gated_case(rng, m, k, n, trans_b=1):
    x = rng.standard_normal((m, k)).astype(np.float16)
    w = [(rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float16) for _ in range(2)]
    return {"x": x, "w_gate": w[0] if trans_b else w[0].T.copy(), "w_up": w[1] if trans_b else w[1].T.copy()}


def gated_result(inputs, activation, trans_b=1):
    """(result, tolerance). Sums of k products: every addition rounds by at
    most 2^-23 of what has been summed, fewer than k / 2 + 16 times in any of
    the orders used (the general form adds one product at a time with half
    that error, the others sixteen and more at once). The activations' fast
    exponential and erf add below 2^-18 relative and 2^-20 |g| absolute."""
    x = inputs["x"].astype(np.float64)
    w = [inputs[name].astype(np.float64) for name in ("w_gate", "w_up")]
    if trans_b:
        w = [a.T for a in w]
    k = x.shape[1]
    g, u = x @ w[0], x @ w[1]
    unit = (k / 2 + 16) * 2.0**-23
    dg, du = (unit * (np.abs(x) @ np.abs(a)) for a in w)
    return _gated(g, u, dg, du, activation)


def _gated(g, u, dg, du, activation):
    a = activate(g, activation)
    y = a * u
    tol = 1.13 * dg * np.abs(u) + (np.abs(a) + 1.13 * dg) * du + np.abs(u) * (2.0**-18 * np.abs(a) + 2.0**-20 * np.abs(g))
    return y, tol + HALF * np.abs(y) + HALF_MIN


def qgemm_case(rng, m, k, n, bias, trans_b=1):
    x, x_scale = quantized(rng, m, k)
    w, w_scale = quantized(rng, n, k)
    inputs = {"x": x, "x_scale": x_scale * 60, "w": w if trans_b else w.T.copy(), "w_scale": w_scale}
    if bias:
        inputs["bias"] = rng.standard_normal(n).astype(np.float16)
    return inputs


def _dequantized(inputs, w_name, s_name, trans_b):
    """x . w with its scales, and its FP32 error: the sum's conversion, the
    scales' product and theirs, half a step each."""
    w = inputs[w_name].astype(np.float64)
    acc = inputs["x"].astype(np.float64) @ (w.T if trans_b else w)
    y = acc * inputs["x_scale"].astype(np.float64)[:, None] * inputs[s_name].astype(np.float64)
    return y, 3 * 2.0**-24 * np.abs(y)


def qgemm_result(inputs, trans_b=1):
    y, tol = _dequantized(inputs, "w", "w_scale", trans_b)
    if "bias" in inputs:
        y = y + inputs["bias"].astype(np.float64)
        tol = tol + 2.0**-24 * np.abs(y)
    return y, tol + HALF * np.abs(y) + HALF_MIN


def qgated_case(rng, m, k, n, trans_b=1):
    x, x_scale = quantized(rng, m, k)
    gate, gate_scale = quantized(rng, n, k)
    up, up_scale = quantized(rng, n, k)
    turn = (lambda a: a) if trans_b else (lambda a: a.T.copy())
    return {"x": x, "x_scale": x_scale * 60, "w_gate": turn(gate), "gate_scale": gate_scale, "w_up": turn(up),
            "up_scale": up_scale}


def qgated_result(inputs, activation, trans_b=1):
    g, dg = _dequantized(inputs, "w_gate", "gate_scale", trans_b)
    u, du = _dequantized(inputs, "w_up", "up_scale", trans_b)
    return _gated(g, u, dg, du, activation)


def quantize_result(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """In 64 bits; a quotient of an 11-bit by a 24-bit value is a half plus or
    minus at least 2^-32 of itself or exactly a half, so rounding its 53-bit
    value rounds it rightly."""
    wide = np.abs(x.astype(np.float64))
    with np.errstate(invalid="ignore", divide="ignore"):
        largest = np.where(np.isnan(wide).any(axis=1), np.nan, wide.max(axis=1))
        scale = (largest / 127.0).astype(np.float32)
        q = np.rint(x.astype(np.float64) / scale.astype(np.float64)[:, None])
    regular = np.isfinite(largest) & (largest > 0)
    q = np.where(regular[:, None], q, 0.0)
    return q.astype(np.int8), scale


def assert_within(actual: np.ndarray, result: tuple[np.ndarray, np.ndarray], what: str) -> None:
    expected, tol = result
    assert actual.shape == expected.shape, (what, actual.shape, expected.shape)
    err = np.abs(actual.astype(np.float64) - expected)
    bad = ~(err <= tol)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, err / tol, 0)), err.shape)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} outside tolerance; worst at {i}: {actual[i]} vs "
                             f"{expected[i]}, tolerance {tol[i]:.3e}")


def gelu_tail_case(rng, op, m, n):
    """Gates from -12 to -0.2 beside `up` projections that bring the products
    back into FP16's normal range: one product a sum, so that gate and up
    are exact in FP32 (in FP16 `up` ends at 65504, and so the gates at -5.8).
    Returns inputs, and gate and up in 64 bits."""
    k = 16
    row = 1 + np.arange(m) % 3 / 64
    if op == "GatedGemm":
        g = -np.exp(rng.uniform(np.log(0.2), np.log(5.6), n)).astype(np.float16).astype(np.float64)
        reach = np.abs(activate_tail(g))
        u = np.minimum(1 / reach, 40000).astype(np.float16).astype(np.float64)
        x, wg, wu = np.zeros((m, k), np.float16), np.zeros((n, k), np.float16), np.zeros((n, k), np.float16)
        x[:, 3], wg[:, 3], wu[:, 3] = row, g, u
        return {"x": x, "w_gate": wg, "w_up": wu}, np.outer(row, g), np.outer(row, u)
    g = -np.exp(rng.uniform(np.log(0.2), np.log(12.0), n))
    x, wg, wu = np.zeros((m, k), np.int8), np.zeros((n, k), np.int8), np.zeros((n, k), np.int8)
    x[:, 5], wg[:, 5], wu[:, 5] = 127, -127, 127
    x_scale = (row / 127).astype(np.float32)
    gate_scale = (-g / 127).astype(np.float32)
    up_scale = (1 / np.abs(activate_tail(g)) / 127).astype(np.float32)
    gate = -127.0 * 127 * np.outer(x_scale.astype(np.float64), gate_scale.astype(np.float64))
    up = 127.0 * 127 * np.outer(x_scale.astype(np.float64), up_scale.astype(np.float64))
    return {"x": x, "x_scale": x_scale, "w_gate": wg, "gate_scale": gate_scale, "w_up": wu, "up_scale": up_scale}, gate, up


def activate_tail(g: np.ndarray) -> np.ndarray:
    """The erf-GELU in 64 bits without cancellation."""
    import math

    return g * 0.5 * np.vectorize(math.erfc)(-g / math.sqrt(2.0))


def gelu_tail_result(gate, up):
    """(result, tolerance), relative throughout. The activation in FP32: 2^-18 +
    g^2 2^-23 (fit 1.43e-6, reciprocal, polynomial and exponential 2^-20 and
    less together; the exponent's roundings grow with it). A gate off by d relative moves GELU by at most (g^2 + 2) d for
    g < 0 (g phi / Phi < g^2 + 1 there): the scales' product and theirs, half a
    step each, 2^-23 in all. The same 2^-23 on up, half a step for the final
    product, and the rounding to FP16."""
    y = activate_tail(gate) * up
    unit = 2.0**-18 + gate**2 * 2.0**-23 + (gate**2 + 2) * 2.0**-23 + 2.0**-23 + 2.0**-24
    return y, np.abs(y) * (unit + HALF) + HALF_MIN
