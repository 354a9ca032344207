"""Measured cases of the feed-forward operators of language models.

Four graph operators are covered: ``GatedGemm`` (gate and up projection,
activation and product in FP16), ``QuantizeRows`` (FP16 rows to 8-bit integers
with one scale a row), ``QGemm`` (8-bit product with a scale for each token and
each output channel) and ``QGatedGemm`` (the gated pair on 8-bit operands).

Where ``own`` is false, :func:`run` computes them with elementary torch
operations in 32 bits; where it is true, it runs the graph that
:func:`prepare` compiled for them. Weights are given as checkpoints store
them, one row for each output channel, and stay on the device.
"""

import functools
import math

import torch

own = False

SILU, GELU = 0, 1


def listed():
    return [
        # One token of a small model: two weight matrices of 8 MB, all latency.
        {"name": "gated-1x1024x4096", "op": "gated", "m": 1, "k": 1024, "n": 4096, "act": SILU},
        # A decode step of sixteen sequences: 201 MB of weights pass once.
        {"name": "gated-16x4096x12288", "op": "gated", "m": 16, "k": 4096, "n": 12288, "act": SILU},
        # A short prompt on a layer whose inner width fits no tile, GELU gate.
        {"name": "gated-333x1008x2731", "op": "gated", "m": 333, "k": 1008, "n": 2731, "act": GELU},
        # A batch of prompts: the largest product in 16 bits.
        {"name": "gated-8192x4096x8192", "op": "gated", "m": 8192, "k": 4096, "n": 8192, "act": SILU},
        # The rows of a decode step before an 8-bit product.
        {"name": "quantize-8x4096", "op": "quantize", "m": 8, "k": 4096},
        # Rows of odd length: neither vectors nor warps divide them.
        {"name": "quantize-4099x5461", "op": "quantize", "m": 4099, "k": 5461},
        # The rows of a long batch: 403 MB in one pass.
        {"name": "quantize-16384x8192", "op": "quantize", "m": 16384, "k": 8192},
        # The down projection of one decode step in 8 bits, with a bias.
        {"name": "qgemm-8x12288x4096", "op": "qgemm", "m": 8, "k": 12288, "n": 4096, "bias": True},
        # A ragged prompt: odd rows and odd output channels.
        {"name": "qgemm-777x2064x1531", "op": "qgemm", "m": 777, "k": 2064, "n": 1531, "bias": False},
        # The down projection of a batch of prompts.
        {"name": "qgemm-8192x8192x4096", "op": "qgemm", "m": 8192, "k": 8192, "n": 4096, "bias": False},
        # A decode step of 32 sequences through an 8-bit gated layer.
        {"name": "qgated-32x4096x12288", "op": "qgated", "m": 32, "k": 4096, "n": 12288, "act": SILU},
        # A prompt of two thousand tokens through the same kind of layer.
        {"name": "qgated-2048x4096x11000", "op": "qgated", "m": 2048, "k": 4096, "n": 11000, "act": GELU},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Tokens from 1 to 16384, hidden widths that are multiples of 16 (every
    width that a product sums over in the field is), any number of output
    channels, rows to quantise of any length."""
    op = rng.choice(["gated", "quantize", "qgemm", "qgated"])
    while True:
        m = _log(rng, 1, 16384)
        if op == "quantize":
            return {"op": op, "m": m, "k": _log(rng, 64, 8192)}
        k = 16 * _log(rng, 16, 768)
        n = _log(rng, 256, 12288)
        if m * k * n <= 8192 * 4096 * 8192:
            break
    if op == "qgemm":
        return {"op": op, "m": m, "k": k, "n": n, "bias": rng.random() < 0.5}
    return {"op": op, "m": m, "k": k, "n": n, "act": rng.choice([SILU, GELU])}


def work(case):
    m, k, n = case["m"], case["k"], case.get("n", 0)
    if case["op"] == "quantize":
        return {"bytes": 3 * m * k + 4 * m, "flops": 2 * m * k}
    if case["op"] == "gated":
        return {"bytes": 2 * (m * k + 2 * k * n + m * n), "flops": 4 * m * k * n}
    if case["op"] == "qgemm":
        return {"bytes": m * k + 4 * m + k * n + 4 * n + 2 * m * n + (2 * n if case["bias"] else 0),
                "flops": 2 * m * k * n}
    return {"bytes": m * k + 4 * m + 2 * (k * n + 4 * n) + 2 * m * n, "flops": 4 * m * k * n}


# ---- inputs -------------------------------------------------------------------


def _activations(gen, m, k):
    """Hidden states as they leave a normalisation: unit variance, a few
    channels many times larger."""
    x = torch.randn(m, k, generator=gen, device="cuda", dtype=torch.float16)
    loud = torch.randint(0, k, (max(1, k // 512),), generator=gen, device="cuda")
    x[:, loud] *= 8.0
    return x


def _weights(gen, n, k):
    return torch.randn(n, k, generator=gen, device="cuda", dtype=torch.float16) / math.sqrt(k)


def _in_8_bits(rows):
    """A matrix quantised symmetrically by rows: what a checkpoint or an
    earlier step holds."""
    scale = rows.abs().amax(dim=1).float() / 127.0
    return torch.round(rows.float() / scale[:, None]).to(torch.int8), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    m, k, n = case["m"], case["k"], case.get("n", 0)
    tensors = {}
    if case["op"] in ("gated", "quantize"):
        tensors["x"] = _activations(gen, m, k)
    else:
        tensors["x"], tensors["x_scale"] = _in_8_bits(_activations(gen, m, k))
    if case["op"] == "gated":
        tensors["w_gate"] = _weights(gen, n, k)
        tensors["w_up"] = _weights(gen, n, k)
    elif case["op"] == "qgemm":
        tensors["w"], tensors["w_scale"] = _in_8_bits(_weights(gen, n, k))
        if case["bias"]:
            tensors["bias"] = torch.randn(n, generator=gen, device="cuda", dtype=torch.float16)
    elif case["op"] == "qgated":
        tensors["w_gate"], tensors["gate_scale"] = _in_8_bits(_weights(gen, n, k))
        tensors["w_up"], tensors["up_scale"] = _in_8_bits(_weights(gen, n, k))
    state = {"case": case, "tensors": tensors}
    if own:
        _compile(state)
    return state


_NODES = {  # operator -> graph node, its inputs in order
    "gated": ("GatedGemm", ("x", "w_gate", "w_up")),
    "quantize": ("QuantizeRows", ("x",)),
    "qgemm": ("QGemm", ("x", "x_scale", "w", "w_scale", "bias")),
    "qgated": ("QGatedGemm", ("x", "x_scale", "w_gate", "gate_scale", "w_up", "up_scale")),
}
_NUMPY = {torch.float16: "float16", torch.float32: "float32", torch.int8: "int8"}


@functools.cache
def _engine(op, names, shapes, dtypes, outputs, attributes):
    """The compiled one-node graph of a case; a program compiles its graph
    once and binds each request's tensors to a context."""
    import cutriton_b200 as ct

    model = ct.Model()
    for name, shape, dtype in zip(names, shapes, dtypes):
        model.add_input(name, list(shape), dtype=dtype, layout="")
    model.add_node("node", op, list(names), list(outputs), **dict(attributes))
    for name in outputs:
        model.add_output(name)
    return ct.build_engine(model, enable_profiling=False, tuning_mode=ct.TUNING_DISABLED)


def _compile(state):
    """A context of the case's graph with the state's tensors bound to its
    inputs and buffers of its own bound to its outputs."""
    case, tensors = state["case"], state["tensors"]
    op_type, names = _NODES[case["op"]]
    names = tuple(name for name in names if name in tensors)
    attributes = {}
    if case["op"] == "quantize":
        outputs = {"q": torch.empty(case["m"], case["k"], dtype=torch.int8, device="cuda"),
                   "q_scale": torch.empty(case["m"], dtype=torch.float32, device="cuda")}
    else:
        outputs = {"y": torch.empty(case["m"], case["n"], dtype=torch.float16, device="cuda")}
        attributes["transB"] = 1
        if "act" in case:
            attributes["activation"] = case["act"]
    engine = _engine(op_type, names, tuple(tuple(tensors[name].shape) for name in names),
                     tuple(_NUMPY[tensors[name].dtype] for name in names), tuple(outputs), tuple(attributes.items()))
    context = engine.create_context()
    for name in names:
        context.bind_tensor(name, tensors[name])
    for name, tensor in outputs.items():
        context.bind_tensor(name, tensor, output=True)
    state["context"] = context
    state["outputs"] = list(outputs.values())


@functools.cache
def _stream():
    """The stream of the program's steps (the legacy default stream cannot be
    captured, so a program of this framework has one), and the events that
    order it with the caller's."""
    return torch.cuda.Stream(), torch.cuda.Event(), torch.cuda.Event()


# ---- one pass -----------------------------------------------------------------


def run(state):
    """Ordered with the current stream as torch's own operations are: the run
    reads what that stream has written, and what follows on it reads the run's
    outputs. An error that a kernel reports is raised by the context's next
    synchronize, the one of the following run at the latest."""
    if own:
        stream, before, after = _stream()
        caller = torch.cuda.current_stream()
        # A context has one run in flight: its last one is taken in first.
        state["context"].synchronize()
        if not caller.query():  # (finished work needs no event)
            before.record(caller)
            stream.wait_event(before)
        state["context"].run_async(stream.cuda_stream)
        after.record(stream)
        caller.wait_event(after)
        return state["outputs"]
    case, t = state["case"], state["tensors"]
    if case["op"] == "gated":
        x = t["x"].float()
        gate = x @ t["w_gate"].float().T
        return [(_activate(gate, case["act"]) * (x @ t["w_up"].float().T)).half()]
    if case["op"] == "quantize":
        return list(_quantize(t["x"]))
    x = t["x"].float()
    if case["op"] == "qgemm":
        y = (x @ t["w"].float().T) * t["x_scale"][:, None] * t["w_scale"]
        return [(y + t["bias"].float() if case["bias"] else y).half()]
    gate = (x @ t["w_gate"].float().T) * t["x_scale"][:, None] * t["gate_scale"]
    up = (x @ t["w_up"].float().T) * t["x_scale"][:, None] * t["up_scale"]
    return [(_activate(gate, case["act"]) * up).half()]


def _activate(gate, act):
    if act == SILU:
        return gate / (1.0 + torch.exp(-gate))
    return 0.5 * gate * (1.0 + torch.erf(gate * math.sqrt(0.5)))


def _quantize(x):
    """Symmetric by rows: scale = max|x| / 127, q = round-half-even(x / scale).
    In 64 bits, since a quotient next to a half decides a whole number."""
    largest = x.abs().amax(dim=1).double()
    scale = (largest / 127.0).float()
    q = torch.round(x.double() / torch.where(scale > 0, scale, 1.0).double()[:, None])
    return q.to(torch.int8), scale


# ---- the definition in 64 bits ------------------------------------------------


def exact(case, seed):
    t = prepare(case, seed)["tensors"]
    with torch.no_grad():
        if case["op"] == "quantize":
            x = t["x"].to(torch.float64)
            scale = torch.maximum(x.max(dim=1).values, -x.min(dim=1).values) / 127
            return [None, scale]
        wide = {name: value.to(torch.float64) for name, value in t.items()}
        if "x_scale" in wide:
            wide["x"] = torch.mul(wide["x"], wide["x_scale"].unsqueeze(1))
        if case["op"] == "qgemm":
            w = torch.mul(wide["w"], wide["w_scale"].unsqueeze(1))
            y = torch.einsum("mk,nk->mn", wide["x"], w)
            return [y.add(wide["bias"]) if case["bias"] else y]
        for name in ("gate", "up"):
            if name + "_scale" in wide:
                wide["w_" + name].mul_(wide[name + "_scale"].unsqueeze(1))
        gate = torch.einsum("mk,nk->mn", wide["x"], wide["w_gate"])
        up = torch.einsum("mk,nk->mn", wide["x"], wide["w_up"])
        if case["act"] == SILU:
            share = torch.tanh(gate / 2).add(1).div(2)
        else:
            share = torch.special.erfc(gate.neg() / math.sqrt(2)).div(2)
        return [gate.mul_(share).mul_(up)]
