"""The gated and 8-bit products and the row quantiser on the GPU, every
candidate against results in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

import cutriton_b200 as ct
import feed_forward_cases as ff

pytestmark = pytest.mark.gpu


class Runner:
    """An engine and a context with CUDA copies of the graph inputs bound; the
    outputs lie inside larger buffers whose edges must stay as they were."""

    GUARD = 64

    def __init__(self, model, inputs, **options):
        import torch

        options.setdefault("enable_cuda_graph", False)
        options.setdefault("tuning_mode", ct.TUNING_DISABLED)
        self.engine = ct.build_engine(model, **options)
        self.context = self.engine.create_context()
        self.inputs = {name: torch.from_numpy(np.ascontiguousarray(a)).cuda() for name, a in inputs.items()}
        for name, t in self.inputs.items():
            self.context.bind_tensor(name, t)
        self.outputs = {}
        self._whole = {}

    def output(self, name, shape, dtype):
        import torch

        dtype = getattr(torch, np.dtype(dtype).name)
        count = int(np.prod(shape))
        size = torch.empty(0, dtype=dtype).element_size()
        # 64 guard elements on both sides; 128 bytes keep the middle aligned.
        guard = max(self.GUARD, 128 // size)
        whole = torch.full((count + 2 * guard,), 77, dtype=dtype, device="cuda")
        self._whole[name] = (whole, guard)
        self.outputs[name] = whole[guard:guard + count].view(shape)
        self.context.bind_tensor(name, self.outputs[name], output=True)

    def run(self, candidate=None):
        import torch

        for t in self.outputs.values():
            t.fill_(77)
        torch.cuda.synchronize()
        if candidate is not None:
            self.context.select_candidate(0, candidate)
        self.context.run()
        for name, (whole, guard) in self._whole.items():
            assert bool((whole[:guard] == 77).all()) and bool((whole[-guard:] == 77).all()), f"{name}: edges written"
        return {name: t.cpu().numpy() for name, t in self.outputs.items()}


def check_product(op, inputs, result, constants=(), **attributes):
    m, n = result[0].shape
    runner = Runner(ff.product_graph(op, inputs, constants, **attributes),
                    {k: v for k, v in inputs.items() if k not in constants})
    runner.output("y", (m, n), np.float16)
    ff.assert_within(runner.run()["y"], result, f"{op} default")
    candidates = runner.engine.op(0)["candidates"]
    for index, name in enumerate(candidates):
        try:
            y = runner.run(index)["y"]
        except ct.CutritonError as error:
            # A form for few rows, pinned where it does not apply.
            assert error.code == ct.SHAPE_ERROR and ("stream" in name or "narrow" in name), (name, error)
            continue
        if name.startswith("unfused"):
            continue  # rounds between its steps; see test_unfused_gated_gemm
        ff.assert_within(y, result, f"{op} {name}")
    return candidates


# Rows, inner and outer sizes around the tiles of every form: single rows and
# columns, the row counts where forms change, sizes that end inside a tile, a
# vector or an 8-element group, and inner sizes of no alignment.
SIZES = [(1, 8, 1), (1, 16, 8), (1, 1024, 300), (2, 64, 9), (5, 136, 257), (8, 1040, 40), (9, 272, 33), (16, 2048, 129),
         (17, 80, 64), (31, 512, 100), (33, 144, 200), (64, 4112, 72), (65, 160, 127), (127, 256, 250),
         (129, 96, 513), (255, 1008, 130), (257, 624, 383), (600, 208, 1000), (3, 7, 5), (70, 33, 90), (130, 1001, 66)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("activation", [ff.SILU, ff.GELU])
def test_gated_gemm(cuda, size, activation):
    inputs = ff.gated_case(np.random.default_rng(size), *size)
    check_product("GatedGemm", inputs, ff.gated_result(inputs, activation), activation=activation, transB=1)


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("bias", [False, True])
def test_qgemm(cuda, size, bias):
    inputs = ff.qgemm_case(np.random.default_rng(size), *size, bias)
    check_product("QGemm", inputs, ff.qgemm_result(inputs), transB=1)


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("activation", [ff.SILU, ff.GELU])
def test_qgated_gemm(cuda, size, activation):
    inputs = ff.qgated_case(np.random.default_rng(size), *size)
    check_product("QGatedGemm", inputs, ff.qgated_result(inputs, activation), activation=activation, transB=1)


# 17 to 64 rows over every split of K: parts without a block of K, widths on both
# sides of each limit and off a tile.
NARROW = [(17, 16, 1), (32, 1040, 1536), (25, 16, 1537), (31, 4112, 2000), (32, 272, 9472), (18, 528, 9473),
          (32, 144, 18945), (33, 2064, 1000), (64, 80, 1600), (63, 6160, 130)]


@pytest.mark.parametrize("op", ["GatedGemm", "QGemm", "QGatedGemm"])
@pytest.mark.parametrize("size", NARROW, ids=lambda s: "x".join(map(str, s)))
def test_narrow_products(cuda, op, size):
    m, k, n = size
    case, result = {"GatedGemm": (ff.gated_case, lambda i: ff.gated_result(i, ff.GELU)),
                    "QGemm": (lambda *a: ff.qgemm_case(*a, True), ff.qgemm_result),
                    "QGatedGemm": (ff.qgated_case, lambda i: ff.qgated_result(i, ff.GELU))}[op]
    inputs = case(np.random.default_rng(size), m, k, n)
    attributes = {"transB": 1, **({} if op == "QGemm" else {"activation": ff.GELU})}
    runner = Runner(ff.product_graph(op, inputs, **attributes), inputs)
    runner.output("y", (m, n), np.float16)
    y = runner.run()["y"]
    name = runner.engine.op(0)["candidates"][runner.context.selected_candidate(0)]
    split = 8 if n <= 1536 else 4 if n <= 9472 else 2 if n <= 18944 else 1
    assert (f".narrow{split}:" in name) == (m <= 32 or (op == "QGemm" and split >= 4)), name
    ff.assert_within(y, result(inputs), name)
    np.testing.assert_array_equal(runner.run()["y"], y)


@pytest.mark.parametrize("constant", [False, True])
@pytest.mark.parametrize("size", [(1, 64, 24), (40, 272, 130), (200, 528, 300)], ids=str)
def test_weights_by_columns(cuda, size, constant):
    """transB = 0, the weights as constants and as graph inputs."""
    rng = np.random.default_rng(7)
    weights = ("w_gate", "w_up", "w") if constant else ()
    inputs = ff.gated_case(rng, *size, trans_b=0)
    check_product("GatedGemm", inputs, ff.gated_result(inputs, 0, trans_b=0), weights)
    inputs = ff.qgemm_case(rng, *size, True, trans_b=0)
    check_product("QGemm", inputs, ff.qgemm_result(inputs, trans_b=0), weights)
    inputs = ff.qgated_case(rng, *size, trans_b=0)
    check_product("QGatedGemm", inputs, ff.qgated_result(inputs, 1, trans_b=0), weights, activation=1)


def test_sums_of_extreme_integers_are_exact(cuda):
    """All products -128 * -128 = 2^14 over the longest inner dimension: the
    sum 131056 * 2^14 fits 32 bits, and 2^-31 of it is exact in FP16."""
    k = 131056
    for m in (1, 130):
        x = np.full((m, k), -128, np.int8)
        w = np.full((40, k), -128, np.int8)
        w[1::2] = 127
        inputs = {"x": x, "x_scale": np.full(m, 2.0**-16, np.float32), "w": w,
                  "w_scale": np.full(40, 2.0**-15, np.float32)}
        check_product("QGemm", inputs, ff.qgemm_result(inputs), transB=1)


def test_large_values_and_non_finite_rows(cuda):
    """Gates far out on both sides, results beyond FP16 (infinite), rows of
    NaN and infinity that leave the other rows alone."""
    rng = np.random.default_rng(3)
    for m in (6, 200):
        inputs = ff.gated_case(rng, m, 128, 70)
        inputs["x"][0] *= np.float16(200)
        inputs["x"][1, 5] = np.nan
        inputs["x"][2, 9] = np.inf
        clean = {**inputs, "x": np.where(np.isfinite(inputs["x"]), inputs["x"], np.float16(0))}
        for activation in (0, 1):
            runner = Runner(ff.product_graph("GatedGemm", inputs, activation=activation, transB=1), inputs)
            runner.output("y", (m, 70), np.float16)
            expected, tol = ff.gated_result(clean, activation)
            for index, name in enumerate(runner.engine.op(0)["candidates"]):
                try:
                    y = runner.run(index)["y"]
                except ct.CutritonError as error:
                    assert error.code == ct.SHAPE_ERROR and ("stream" in name or "narrow" in name)
                    continue
                assert np.isnan(y[1]).all() and not np.isfinite(y[2]).any(), name
                over = np.abs(expected) > 65600
                assert np.isinf(y[0][over[0]]).all(), name
                inside = (np.abs(expected) < 65000) & ~np.isin(np.arange(m), (1, 2))[:, None]
                if not name.startswith("unfused"):
                    assert (np.abs(y.astype(np.float64) - expected) <= tol)[inside].all(), name
        q = ff.qgemm_case(rng, m, 128, 70, False)
        q["x_scale"][1], q["x_scale"][2] = np.nan, np.inf
        q["x"][2] = 0  # what QuantizeRows gives for a row with an infinity
        runner = Runner(ff.product_graph("QGemm", q, transB=1), q)
        runner.output("y", (m, 70), np.float16)
        y = runner.run()["y"]
        assert np.isnan(y[1]).all() and np.isnan(y[2]).all()
        assert np.isfinite(y[[0, *range(3, m)]]).all()


@pytest.mark.parametrize("rows", [5, 150])
@pytest.mark.parametrize("activation", [ff.SILU, ff.GELU])
def test_non_finite_weights_stay_in_their_column(cuda, activation, rows):
    """NaN or infinities in single output channels; gates far out on the side
    where the activation vanishes, next to ordinary ones."""
    inputs = ff.gated_case(np.random.default_rng(13), rows, 96, 76)
    inputs["x"] = np.abs(inputs["x"]) + np.float16(0.5)
    bad = {3: np.nan, 10: np.inf, 11: -np.inf, 40: np.nan, 73: np.nan}
    inputs["w_gate"][20] = -60000
    inputs["w_gate"][21] = 60000
    inputs["w_gate"][75] = -1
    clean = {n: a.copy() for n, a in inputs.items()}
    for column, value in bad.items():
        inputs["w_gate" if column < 40 else "w_up"][column, column % 7] = value
    expected, tol = ff.gated_result(clean, activation)
    runner = Runner(ff.product_graph("GatedGemm", inputs, activation=activation, transB=1), inputs)
    runner.output("y", (rows, 76), np.float16)
    good = np.setdiff1d(np.arange(76), list(bad))
    for index, name in enumerate(runner.engine.op(0)["candidates"]):
        try:
            y = runner.run(index)["y"]
        except ct.CutritonError as error:
            assert error.code == ct.SHAPE_ERROR and ("stream" in name or "narrow" in name)
            continue
        inside = good[np.abs(expected[:, good]).max(axis=0) < 65000]
        assert (np.abs(y[:, inside].astype(np.float64) - expected[:, inside]) <= tol[:, inside]).all(), name
        assert inside.size >= 65 and not np.isfinite(y[:, [3, 40, 73]]).any(), name


@pytest.mark.parametrize("activation", [ff.SILU, ff.GELU])
def test_unfused_gated_gemm(cuda, activation):
    """The decomposition rounds gate, activation and up projection to FP16
    too: three more half steps on the product, and theirs on gate and up."""
    inputs = ff.gated_case(np.random.default_rng(5), 70, 200, 90, trans_b=0)
    expected, tol = ff.gated_result(inputs, activation, trans_b=0)
    x = inputs["x"].astype(np.float64)
    g, u = (np.abs(x @ inputs[w].astype(np.float64)) for w in ("w_gate", "w_up"))
    tol = tol + ff.HALF * (1.13 * g * u * (1 + ff.HALF) + 3 * np.abs(expected)) + ff.HALF_MIN * (2 * u + 2)
    runner = Runner(ff.product_graph("GatedGemm", inputs, ("w_gate", "w_up"), activation=activation),
                    {"x": inputs["x"]})
    runner.output("y", (70, 90), np.float16)
    names = runner.engine.op(0)["candidates"]
    ff.assert_within(runner.run(names.index("unfused:gated_gemm"))["y"], (expected, tol), "unfused")


@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (2, 63), (5, 255), (17, 1023), (4, 1024), (9, 1025),
                                   (1, 4096), (6, 5461), (3, 8192), (2, 8193), (2, 20001), (3000, 40), (2500, 1500)], ids=str)
def test_quantize_rows(cuda, shape):
    rng = np.random.default_rng(shape)
    x = (rng.standard_normal(shape) * np.exp(rng.uniform(-12, 8, (shape[0], 1)))).astype(np.float16)
    x[rng.integers(0, shape[0])] = 0
    check_quantize(x)


def check_quantize(x, **options):
    runner = Runner(ff.product_graph("QuantizeRows", {"x": x}), {"x": x}, **options)
    runner.output("q", x.shape, np.int8)
    runner.output("q_scale", x.shape[:1], np.float32)
    got = runner.run()
    q, scale = ff.quantize_result(x)
    np.testing.assert_array_equal(got["q_scale"], scale)
    np.testing.assert_array_equal(got["q"], q)


@pytest.mark.parametrize("shape", [(1, 36864), (3, 36871), (149, 12289), (2, 65529), (301, 40000), (2, 73728), (3, 73730)],
                         ids=str)
def test_quantize_long_rows(cuda, shape):
    """Eight and sixteen warps a row, one or two rows in their queues, and rows
    that no queue holds."""
    x = np.random.default_rng(shape).standard_normal(shape).astype(np.float16)
    x[-1, -1] = 30.0
    check_quantize(x)


def test_quantize_rows_ties_and_special_values(cuda):
    """Scales that are powers of two put quotients exactly on halves; FP16's
    smallest numbers; quotients next to a half; rows of infinity and NaN."""
    x = np.zeros((40, 300), np.float16)
    halves = np.arange(-126.5, 127, 1.0)
    for row in range(20):
        scale = 2.0 ** (row - 17)
        x[row, :halves.size] = halves * scale
        x[row, 299] = 127 * scale
    x[20, :] = np.float16(2.0**-24) * np.arange(300)
    x[21, 3] = np.inf
    x[22, 4] = -np.inf
    x[23, 5] = np.nan
    x[24, 6], x[24, 7] = np.nan, np.inf
    x[25, :] = -0.0
    x[26, 8] = np.float16(2.0**-24)
    x[27, :] = 65504
    rng = np.random.default_rng(0)
    x[28:] = rng.integers(-2047, 2048, (12, 300)).astype(np.float16)
    check_quantize(x)


def test_quantize_every_half_against_every_scale_step(cuda):
    """Every finite FP16 magnitude next to 512 different row maxima."""
    finite = np.arange(0x7C00, dtype=np.uint16).view(np.float16)
    largest = finite[0x3C00:0x3C00 + 512]  # 1.0 ... 1.5: every mantissa of one binade
    below = finite[finite <= 1]
    x = np.concatenate([np.tile(below, (512, 1)), largest[:, None]], axis=1)
    check_quantize(x)


def test_unaligned_tensors(cuda):
    """Graph inputs and outputs that start one element off every alignment."""
    import torch

    rng = np.random.default_rng(11)
    x = rng.standard_normal((5, 2050)).astype(np.float16)
    engine = ct.build_engine(ff.product_graph("QuantizeRows", {"x": x}), tuning_mode=ct.TUNING_DISABLED)
    context = engine.create_context()
    device = torch.zeros(x.size + 1, dtype=torch.float16, device="cuda")
    device[1:] = torch.from_numpy(x).cuda().reshape(-1)
    q = torch.full((x.size + 3,), 77, dtype=torch.int8, device="cuda")
    scale = torch.empty(5, dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    context.bind_tensor("x", device[1:])
    context.bind_tensor("q", q[1:x.size + 1], output=True)
    context.bind_tensor("q_scale", scale, output=True)
    context.run()
    want_q, want_scale = ff.quantize_result(x)
    np.testing.assert_array_equal(q[1:x.size + 1].cpu().numpy().reshape(x.shape), want_q)
    np.testing.assert_array_equal(scale.cpu().numpy(), want_scale)
    assert q[0] == 77 and (q[x.size + 1:] == 77).all()


def test_quantize_rows_every_maximum(cuda):
    """Every finite FP16 magnitude as a row's largest: the scale is the
    rounded quotient for each."""
    x = np.zeros((0x7C00, 12), np.float16)
    x[:, 5] = np.arange(0x7C00, dtype=np.uint16).view(np.float16)
    x[:, 7] = -x[:, 5] / 2
    check_quantize(x)


def single(op, inputs, constants=(), **attributes):
    """The outputs of one node run by itself, on the device."""
    import torch

    engine = ct.build_engine(ff.product_graph(op, {**{n: _host(t) for n, t in inputs.items()}}, constants, **attributes),
                             tuning_mode=ct.TUNING_DISABLED)
    context = engine.create_context()
    for name, tensor in inputs.items():
        if name not in constants:
            context.bind_tensor(name, tensor)
    names = ["q", "q_scale"] if op == "QuantizeRows" else ["y"]
    outputs = []
    for name in names:
        code, shape = engine.value_desc(name)
        dtype = {ct.FLOAT16: torch.float16, ct.FLOAT32: torch.float32, ct.INT8: torch.int8}[code]
        outputs.append(torch.empty(shape, dtype=dtype, device="cuda"))
        context.bind_tensor(name, outputs[-1], output=True)
    torch.cuda.synchronize()
    context.run()
    return outputs


def _host(tensor):
    return tensor if isinstance(tensor, np.ndarray) else tensor.cpu().numpy()


def run_block(model, x, candidates=None, **options):
    import torch

    engine = ct.build_engine(model, tuning_mode=ct.TUNING_DISABLED, **options)
    context = engine.create_context()
    context.bind_tensor("x", x)
    y = torch.full_like(x, 77)
    context.bind_tensor("output", y, output=True)
    torch.cuda.synchronize()
    context.run()
    return y, engine, context


@pytest.mark.parametrize("tokens", [1, 16, 17, 300])
def test_8bit_block_is_its_steps(cuda, tokens):
    """Quantise, gated product, quantise, down projection, residual and norm in
    one graph: bit for bit what the operators give one after another."""
    import torch

    from cutriton_b200 import workloads

    weights = workloads.gated_ffn_weights(192, 528, seed=2)
    x = torch.from_numpy(workloads.ffn_input(tokens, 192, seed=3)).cuda()
    y, _, _ = run_block(workloads.build_gated_ffn_int8(weights, tokens), x)
    eight = {name: workloads.quantize_weight(weights["w_" + name]) for name in ("gate", "up", "down")}
    dev = {f"{n}{i}": torch.from_numpy(a).cuda() for n, pair in eight.items() for i, a in enumerate(pair)}
    x8, x_scale = single("QuantizeRows", {"x": x})
    (h,) = single("QGatedGemm", {"x": x8, "x_scale": x_scale, "w_gate": dev["gate0"], "gate_scale": dev["gate1"],
                                 "w_up": dev["up0"], "up_scale": dev["up1"]}, transB=1)
    h8, h_scale = single("QuantizeRows", {"x": h})
    (down,) = single("QGemm", {"x": h8, "x_scale": h_scale, "w": dev["down0"], "w_scale": dev["down1"]}, transB=1)
    gamma, beta = (torch.from_numpy(weights[n]).cuda() for n in ("gamma", "beta"))
    (want,) = single("SkipLayerNormalization", {"a": down, "x": x, "gamma": gamma, "beta": beta}, epsilon=1e-5, axis=-1)
    assert torch.equal(y, want)


@pytest.mark.parametrize("activation", ["Silu", "Gelu"])
@pytest.mark.parametrize("tokens", [3, 130])
def test_gated_block_is_its_steps(cuda, tokens, activation):
    import torch

    from cutriton_b200 import workloads

    weights = workloads.gated_ffn_weights(128, 336, seed=4)
    x = torch.from_numpy(workloads.ffn_input(tokens, 128, seed=5)).cuda()
    y, engine, _ = run_block(workloads.build_gated_ffn(weights, tokens, activation), x)
    assert engine.op(0)["op_type"] == "GatedGemm"
    constants = {"x": x, "w_gate": weights["w_gate"], "w_up": weights["w_up"]}
    (h,) = single("GatedGemm", constants, ("w_gate", "w_up"), activation=0 if activation == "Silu" else 1)
    (down,) = single("Gemm", {"x": h, "w": weights["w_down"]}, ("w",))
    gamma, beta = (torch.from_numpy(weights[n]).cuda() for n in ("gamma", "beta"))
    (want,) = single("SkipLayerNormalization", {"a": down, "x": x, "gamma": gamma, "beta": beta}, epsilon=1e-5, axis=-1)
    assert torch.equal(y, want)


def test_row_counts_of_one_profile_choose_their_form(cuda):
    """One engine over 1 to 400 tokens: each run equals a static engine of its
    shape, at most 16 rows take the few-row form, captured graphs are kept."""
    import torch

    from cutriton_b200 import workloads

    weights = workloads.gated_ffn_weights(128, 272, seed=6)
    model = workloads.build_gated_ffn_int8(weights, -1)
    model.add_shape_profile("tokens", "x", [1, 128], [64, 128], [400, 128])
    engine = ct.build_engine(model, tuning_mode=ct.TUNING_DISABLED)
    context = engine.create_context()
    ops = engine.ops()
    gated = [o["op_type"] for o in ops].index("QGatedGemm")
    for tokens in (64, 1, 16, 17, 400, 16, 1):
        x = torch.from_numpy(workloads.ffn_input(tokens, 128, seed=tokens)).cuda()
        y = torch.empty_like(x)
        context.set_input_shape("x", [tokens, 128])
        context.resolve_shapes()
        context.bind_tensor("x", x)
        context.bind_tensor("output", y, output=True)
        torch.cuda.synchronize()
        context.run()
        chosen = ops[gated]["candidates"][context.selected_candidate(gated)]
        assert (".stream:" in chosen) == (tokens <= 16), (tokens, chosen)
        want, _, _ = run_block(workloads.build_gated_ffn_int8(weights, tokens), x)
        assert torch.equal(y, want), tokens
    assert context.cached_graph_count() >= 2


def test_replays_and_streams_give_the_same(cuda):
    """A captured graph replayed on changed inputs, two contexts of one engine
    at once on two streams, and a run without graphs."""
    import torch

    from cutriton_b200 import workloads

    weights = workloads.gated_ffn_weights(256, 624, seed=8)
    for tokens in (9, 200):
        xs = [torch.from_numpy(workloads.ffn_input(tokens, 256, seed=s)).cuda() for s in range(6)]
        engine = ct.build_engine(workloads.build_gated_ffn_int8(weights, tokens), tuning_mode=ct.TUNING_DISABLED)
        contexts = [engine.create_context() for _ in range(2)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        bound = [(torch.empty_like(xs[0]), torch.empty_like(xs[0])) for _ in range(2)]
        for context, (x, y) in zip(contexts, bound):
            context.bind_tensor("x", x)
            context.bind_tensor("output", y, output=True)
        got = []
        for i in range(0, 6, 2):
            for j in range(2):
                bound[j][0].copy_(xs[i + j])
            torch.cuda.synchronize()
            for j in range(2):
                contexts[j].run_async(streams[j].cuda_stream)
            for j in range(2):
                contexts[j].synchronize()
                got.append(bound[j][1].clone())
        for x, y in zip(xs, got):
            want, _, _ = run_block(workloads.build_gated_ffn_int8(weights, tokens), x, enable_cuda_graph=0)
            assert torch.equal(y, want)


@pytest.mark.parametrize("eight", [False, True])
def test_narrow_products_between_other_kernels(cuda, eight):
    """Blocks of 24 rows without profiling, so that their kernels start before
    those in front end, on two streams at once: the results of single runs."""
    import torch

    from cutriton_b200 import workloads

    build = workloads.build_gated_ffn_int8 if eight else workloads.build_gated_ffn
    model = build(workloads.gated_ffn_weights(256, 2000, seed=9), 24)
    engine = ct.build_engine(model, tuning_mode=ct.TUNING_DISABLED, enable_profiling=False)
    contexts = [engine.create_context() for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [torch.from_numpy(workloads.ffn_input(24, 256, seed=s)).cuda() for s in range(2)]
    ys = [torch.empty_like(x) for x in xs]
    wants = []
    for context, x, y in zip(contexts, xs, ys):
        context.bind_tensor("x", x)
        context.bind_tensor("output", y, output=True)
        torch.cuda.synchronize()
        context.run()
        wants.append(y.clone())
    names = [op["candidates"][contexts[0].selected_candidate(i)] for i, op in enumerate(engine.ops())]
    assert any(".narrow4:" in name for name in names), names
    for _ in range(20):
        for y in ys:
            y.zero_()
        torch.cuda.synchronize()
        for context, stream in zip(contexts, streams):
            context.run_async(stream.cuda_stream)
        for context in contexts:
            context.synchronize()
        for y, want in zip(ys, wants):
            assert torch.equal(y, want)


@pytest.mark.parametrize("rows", [4, 40])
def test_tuner_chooses_among_the_forms_that_take_the_shape(cuda, tmp_path, rows):
    rng = np.random.default_rng(9)
    inputs = ff.qgemm_case(rng, rows, 256, 96, True)
    runner = Runner(ff.product_graph("QGemm", inputs, transB=1), inputs, tuning_mode=ct.TUNING_TUNE_ON_MISS,
                    tuning_cache_dir=str(tmp_path))
    runner.output("y", (rows, 96), np.float16)
    ff.assert_within(runner.run()["y"], ff.qgemm_result(inputs), "tuned")
    chosen = runner.engine.op(0)["candidates"][runner.context.selected_candidate(0)]
    assert rows <= 16 or ".stream:" not in chosen
    assert len(list(tmp_path.glob("*.json"))) == 1


def test_facade_runs_the_8bit_pair(cuda, tmp_path):
    import json

    from cutriton_b200 import api

    rng = np.random.default_rng(10)
    w, scale = ff.quantized(rng, 24, 48)
    graph = {"inputs": ["x"], "outputs": ["x8", "xs", "y"], "input_dtypes": {"x": "float16"},
             "nodes": [{"name": "q", "op_type": "QuantizeRows", "inputs": ["x"], "outputs": ["x8", "xs"]},
                       {"name": "p", "op_type": "QGemm", "inputs": ["x8", "xs", "w", "ws"], "outputs": ["y"],
                        "transB": 1}],
             "constants": {"w": {"data": w.ravel().tolist(), "shape": [24, 48], "dtype": "int8"},
                           "ws": {"data": scale.tolist(), "shape": [24], "dtype": "float32"}}}
    path = tmp_path / "g.json"
    path.write_text(json.dumps(graph))
    context = api.compile(path).create_context()
    for rows in (2, 30):
        x = rng.standard_normal((rows, 48)).astype(np.float16)
        got = context.run({"x": x})
        q, q_scale = ff.quantize_result(x)
        np.testing.assert_array_equal(got["x8"], q)
        np.testing.assert_array_equal(got["xs"], q_scale)
        ff.assert_within(got["y"], ff.qgemm_result({"x": q, "x_scale": q_scale, "w": w, "w_scale": scale}), "facade")


@pytest.mark.parametrize("rows", [3, 50])
def test_products_off_16_bytes_fail_with_an_error(cuda, rows):
    """An activation bound off 16 bytes: an error, and the context goes on."""
    import torch

    rng = np.random.default_rng(12)
    inputs = ff.gated_case(rng, rows, 64, 40)
    engine = ct.build_engine(ff.product_graph("GatedGemm", inputs, transB=1), tuning_mode=ct.TUNING_DISABLED,
                             enable_cuda_graph=0)
    context = engine.create_context()
    device = {n: torch.from_numpy(a).cuda() for n, a in inputs.items()}
    shifted = torch.zeros(rows * 64 + 1, dtype=torch.float16, device="cuda")
    shifted[1:] = device["x"].reshape(-1)
    y = torch.empty(rows, 40, dtype=torch.float16, device="cuda")
    for name in ("w_gate", "w_up"):
        context.bind_tensor(name, device[name])
    context.bind_tensor("x", shifted[1:])
    context.bind_tensor("y", y, output=True)
    torch.cuda.synchronize()
    with pytest.raises(ct.CutritonError) as error:
        context.run()
    assert error.value.code == ct.RUNTIME_ERROR
    context.bind_tensor("x", device["x"])
    context.run()
    ff.assert_within(y.cpu().numpy(), ff.gated_result(inputs, 0), "after the error")


@pytest.mark.parametrize("shape", [(1, 5), (33, 250), (700, 1000)], ids=str)
def test_silu_and_mul(cuda, shape):
    """The unfused steps: SiLU in FP32 (2^-18 relative for the exponential and
    the division) rounded once, the product in FP16 as numpy's."""
    rng = np.random.default_rng(shape)
    x = (rng.standard_normal(shape) * 8).astype(np.float16)
    x.flat[:5] = [0, -0.0, 65504, -65504, 2.0**-24]
    y = rng.standard_normal(shape).astype(np.float16)
    model = ct.Model()
    for name in "xy":
        model.add_input(name, list(shape), dtype=np.float16, layout="")
    model.add_node("silu", "Silu", ["x"], ["s"])
    model.add_node("mul", "Mul", ["x", "y"], ["m"])
    model.add_output("s")
    model.add_output("m")
    runner = Runner(model, {"x": x, "y": y})
    runner.output("s", shape, np.float16)
    runner.output("m", shape, np.float16)
    got = runner.run()
    want = ff.activate(x.astype(np.float64), ff.SILU)
    tol = (2.0**-18 + ff.HALF) * np.abs(want) + ff.HALF_MIN
    assert (np.abs(got["s"].astype(np.float64) - want) <= tol).all()
    np.testing.assert_array_equal(got["m"], x * y)


def test_offsets_past_32_bits(cuda):
    """More than 2^31 elements in a quantised matrix and in a product's output."""
    import torch

    rows, columns = 524300, 4097
    x = torch.empty(rows, columns, dtype=torch.float16, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    q, scale = single_on_device("QuantizeRows", {"x": x})
    for part in (slice(0, 3), slice(rows // 2, rows // 2 + 3), slice(rows - 3, rows)):
        want_q, want_scale = ff.quantize_result(x[part].cpu().numpy())
        np.testing.assert_array_equal(q[part].cpu().numpy(), want_q)
        np.testing.assert_array_equal(scale[part].cpu().numpy(), want_scale)
    del x, q, scale
    m, n, k = 70001, 32769, 48
    rng = np.random.default_rng(2)
    inputs = ff.gated_case(rng, m, k, n)
    (y,) = single_on_device("GatedGemm", {name: torch.from_numpy(a).cuda() for name, a in inputs.items()}, transB=1)
    for part in (slice(0, 2), slice(m // 2, m // 2 + 2), slice(m - 2, m)):
        ff.assert_within(y[part].cpu().numpy(), ff.gated_result({**inputs, "x": inputs["x"][part]}, 0), "far rows")


@pytest.mark.parametrize("op", ["GatedGemm", "QGemm", "QGatedGemm"])
def test_more_columns_than_a_grid_dimension_of_tiles(cuda, op):
    """The general form (odd K) over 65538 tiles of 64 columns, both ways round."""
    import torch

    wide = 65536 * 64 + 70
    for m, n in ((2, wide), (wide, 2)):
        rng = np.random.default_rng(21)
        case, result = {"GatedGemm": (ff.gated_case, lambda i: ff.gated_result(i, ff.SILU)),
                        "QGemm": (lambda *a: ff.qgemm_case(*a, True), ff.qgemm_result),
                        "QGatedGemm": (ff.qgated_case, lambda i: ff.qgated_result(i, ff.SILU))}[op]
        inputs = case(rng, m, 3, n)
        (y,) = single_on_device(op, {name: torch.from_numpy(a).cuda() for name, a in inputs.items()}, transB=1)
        ff.assert_within(y.cpu().numpy(), result(inputs), f"{m}x{n}")


def single_on_device(op, tensors, **attributes):
    """One node over device tensors, without host copies of them."""
    import torch

    names = {torch.float16: "float16", torch.int8: "int8", torch.float32: "float32"}
    model = ct.Model()
    for name, t in tensors.items():
        model.add_input(name, list(t.shape), dtype=names[t.dtype], layout="")
    outs = ["q", "q_scale"] if op == "QuantizeRows" else ["y"]
    model.add_node("node", op, list(tensors), outs, **attributes)
    for name in outs:
        model.add_output(name)
    engine = ct.build_engine(model, tuning_mode=ct.TUNING_DISABLED)
    context = engine.create_context()
    for name, t in tensors.items():
        context.bind_tensor(name, t)
    outputs = []
    for name in outs:
        code, shape = engine.value_desc(name)
        dtype = {ct.FLOAT16: torch.float16, ct.FLOAT32: torch.float32, ct.INT8: torch.int8}[code]
        outputs.append(torch.empty(shape, dtype=dtype, device="cuda"))
        context.bind_tensor(name, outputs[-1], output=True)
    torch.cuda.synchronize()
    context.run()
    return outputs


@pytest.mark.parametrize("op", ["GatedGemm", "QGemm", "QGatedGemm"])
def test_pairs_whose_second_half_has_no_rows(cuda, op):
    """One or two blocks of K, one or two tiles a pair and rows for one CTA of it
    only: its peer has arrived on all of its barriers before it leaves. Forty
    runs one behind the other, all alike."""
    case, result = {"GatedGemm": (ff.gated_case, lambda i: ff.gated_result(i, ff.SILU)),
                    "QGemm": (lambda *a: ff.qgemm_case(*a, True), ff.qgemm_result),
                    "QGatedGemm": (ff.qgated_case, lambda i: ff.qgated_result(i, ff.SILU))}[op]
    for m, k, n in ((1, 16, 8), (33, 144, 40), (129, 16, 4800)):
        inputs = case(np.random.default_rng((m, k, n)), m, k, n)
        runner = Runner(ff.product_graph(op, inputs, transB=1), inputs, enable_profiling=False)
        runner.output("y", (m, n), np.float16)
        (pair,) = [i for i, c in enumerate(runner.engine.op(0)["candidates"]) if ".pair:" in c]
        y = runner.run(pair)["y"]
        ff.assert_within(y, result(inputs), f"{op} {m}x{k}x{n}")
        for _ in range(40):
            runner.context.run()
        np.testing.assert_array_equal(runner.outputs["y"].cpu().numpy(), y)


@pytest.mark.parametrize("op", ["GatedGemm", "QGatedGemm"])
@pytest.mark.parametrize("rows", [1, 12, 24, 150])
def test_gelu_far_below_zero(cuda, op, rows):
    """Every form (few rows, narrow, pairs, general) keeps the small values of
    GELU to FP16's precision where a large up projection shows them."""
    inputs, gate, up = ff.gelu_tail_case(np.random.default_rng(rows), op, rows, 700)
    candidates = check_product(op, inputs, ff.gelu_tail_result(gate, up), activation=ff.GELU, transB=1)
    assert any(".any:" in c for c in candidates)


@pytest.mark.parametrize("activation", [ff.SILU, ff.GELU])
def test_a_token_does_not_depend_on_its_batch(cuda, activation):
    """8-bit sums are exact and every form has the same epilogue arithmetic: a
    row's results are the same bits in a batch of any size and in any form."""
    rng = np.random.default_rng(31)
    inputs = ff.qgated_case(rng, 300, 64, 9000)
    whole = None
    for rows in (300, 60, 24, 12, 1):
        part = {n: a[:rows] if n in ("x", "x_scale") else a for n, a in inputs.items()}
        runner = Runner(ff.product_graph("QGatedGemm", part, activation=activation, transB=1), part)
        runner.output("y", (rows, 9000), np.float16)
        for index, name in enumerate(runner.engine.op(0)["candidates"]):
            try:
                y = runner.run(index)["y"].view(np.uint16)
            except ct.CutritonError as error:
                assert error.code == ct.SHAPE_ERROR and ("stream" in name or "narrow" in name), (name, error)
                continue
            whole = y if whole is None else whole
            assert np.array_equal(y, whole[:rows]), (rows, name, int((y != whole[:rows]).sum()))


@pytest.mark.parametrize("rows", [4, 40])
def test_tuner_skips_a_candidate_that_cannot_be_launched(cuda, tmp_path, rows):
    """A pack whose general form binds a tensor map of the wrong rank: the host
    refuses every launch of it, and tuning goes on among the others. Pinned, it
    is the run's error."""
    import json
    import shutil
    from pathlib import Path

    pack = json.loads((Path(ct.PACK_DIR) / "pack.json").read_text())
    pack["kernels"] = [k for k in pack["kernels"] if k["op_type"] == "QGemm"]
    for kernel in pack["kernels"]:
        target = tmp_path / "pack" / kernel["binary"]
        target.parent.mkdir(parents=True, exist_ok=True)
        shutil.copy(Path(ct.PACK_DIR) / kernel["binary"], target)
        if kernel["kernel_id"] == "qgemm.i8.any":
            kernel["arguments"][0] = {"name": "x", "type": "tensormap", "source": {
                "kind": "tensor_map", "tensor": "input", "index": 0, "box": [32], "swizzle": 0}}
    (tmp_path / "pack" / "pack.json").write_text(json.dumps(pack))
    inputs = ff.qgemm_case(np.random.default_rng(14), rows, 256, 96, True)
    runner = Runner(ff.product_graph("QGemm", inputs, transB=1), inputs, tuning_mode=ct.TUNING_TUNE_ON_MISS,
                    tuning_cache_dir=str(tmp_path / "cache"), kernel_artifact_dir=str(tmp_path / "pack"))
    runner.output("y", (rows, 96), np.float16)
    ff.assert_within(runner.run()["y"], ff.qgemm_result(inputs), "tuned")
    names = runner.engine.op(0)["candidates"]
    (general,) = [i for i, name in enumerate(names) if ".any:" in name]
    assert runner.context.selected_candidate(0) != general
    (choice,) = (tmp_path / "cache").glob("*.json")
    medians = json.loads(choice.read_text())["median_ms"]
    assert medians[names[general]] is None and sum(m is not None for m in medians.values()) >= 2
    with pytest.raises(ct.CutritonError) as error:
        runner.run(general)
    assert error.value.code == ct.SHAPE_ERROR


@pytest.mark.parametrize("from_steps", [False, True])
def test_tuning_keeps_the_definition_of_a_gated_product(cuda, tmp_path, from_steps):
    """K = 203 leaves the general form and the steps. A node written as one op
    has one rounding, whatever is faster; the graph's own steps may run as such."""
    import json

    rng = np.random.default_rng(15)
    inputs = ff.gated_case(rng, 200, 203, 256, trans_b=0)
    weights = ("w_gate", "w_up")
    model = ff.product_graph("GatedGemm", inputs, weights)
    if from_steps:
        model = ct.Model()
        model.add_input("x", [200, 203], dtype=np.float16, layout="")
        for name in weights:
            model.add_constant(name, inputs[name], layout="")
        model.add_node("gate", "Gemm", ["x", "w_gate"], ["g"])
        model.add_node("act", "Silu", ["g"], ["a"])
        model.add_node("up", "Gemm", ["x", "w_up"], ["u"])
        model.add_node("product", "Mul", ["a", "u"], ["y"])
        model.add_output("y")
    runner = Runner(model, {"x": inputs["x"]}, tuning_mode=ct.TUNING_TUNE_ON_MISS, tuning_cache_dir=str(tmp_path))
    runner.output("y", (200, 256), np.float16)
    y = runner.run()["y"]
    (op,) = runner.engine.ops()
    assert op["op_type"] == "GatedGemm" and len(op["candidates"]) == 2
    (choice,) = tmp_path.glob("*.json")
    medians = json.loads(choice.read_text())["median_ms"]
    assert (medians["unfused:gated_gemm"] is not None) == from_steps
    if not from_steps:
        ff.assert_within(y, ff.gated_result(inputs, ff.SILU, trans_b=0), "tuned")
    runner.run(op["candidates"].index("unfused:gated_gemm"))


@pytest.mark.parametrize("rows", [4, 20, 70])
def test_inner_sizes_of_one_profile_choose_their_form(cuda, rows):
    """A profile that leaves K open: lengths that are no whole 16-byte rows take
    the general form, the others the one of their row count."""
    import torch

    model = ct.Model()
    shapes = {"x": (np.int8, lambda k: [rows, k]), "x_scale": (np.float32, lambda k: [rows]),
              "w": (np.int8, lambda k: [24, k]), "w_scale": (np.float32, lambda k: [24])}
    for name, (dtype, shape) in shapes.items():
        model.add_input(name, shape(-1), dtype=dtype, layout="")
    model.add_node("node", "QGemm", list(shapes), ["y"], transB=1)
    model.add_output("y")
    for name, (_, shape) in shapes.items():
        model.add_shape_profile("inner", name, shape(16), shape(64), shape(300))
    engine = ct.build_engine(model, tuning_mode=ct.TUNING_DISABLED)
    context = engine.create_context()
    for k in (64, 17, 300, 272, 18, 16):
        inputs = ff.qgemm_case(np.random.default_rng(k), rows, k, 24, False)
        for name, (_, shape) in shapes.items():
            context.set_input_shape(name, shape(k))
        context.resolve_shapes()
        device = {name: torch.from_numpy(a).cuda() for name, a in inputs.items()}
        y = torch.empty(rows, 24, dtype=torch.float16, device="cuda")
        for name, tensor in device.items():
            context.bind_tensor(name, tensor)
        context.bind_tensor("y", y, output=True)
        torch.cuda.synchronize()
        context.run()
        ff.assert_within(y.cpu().numpy(), ff.qgemm_result(inputs), f"{rows}x{k}")
        chosen = engine.op(0)["candidates"][context.selected_candidate(0)]
        assert (".any:" in chosen) == (k % 16 != 0), (k, chosen)
