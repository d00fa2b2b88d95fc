"""Operators in 8-bit floating point against their definition in 64 bits (plain_fp8): rows, products, feed-forwards, layers of routed experts."""
import pytest
import torch

import plain_fp8 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(key) % (1 << 31))


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _whole(g, *shape, most=4):
    """Whole numbers: their products and sums are exact in float, and none of eight products is 2^-13 of another."""
    return torch.randint(-most, most + 1, shape, generator=g, device=DEV).float()


def _same(got, want):
    """Equal numbers, NaN beside NaN."""
    return bool(((got == want) | (got.isnan() & want.isnan())).all())


def _rows_check(x, q, want_x):
    codes, e = plain.quantised(want_x)
    M, K = want_x.shape
    B = -(-K // 128)
    assert q.shape == (M, K) and q.codes.dtype == F8 and tuple(q.codes.shape) == (M, B * 128)
    assert torch.equal(q.scales[:, :B].int() - 127, e.int())
    assert (q.scales[:, B:] == 127).all()
    assert _same(q.codes.double(), codes)
    assert _same(q.values(), plain.values(codes, e, K).float())       # (256 x 2^120 and more is an infinity in float)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 5120), (3, 127), (5, 128), (2, 129), (17, 511), (64, 640), (33, 1403), (2049, 1032)])
def test_rows_have_the_definitions_codes(M, K, dtype):
    from sharpinference_amd import ops
    g = _gen(M, K)
    x = (_normal(g, M, K) * torch.exp(6 * _normal(g, M, 1))).to(dtype)
    _rows_check(x, ops.quantize_rows(x), x)


def test_every_bfloat16_value_beside_every_largest():
    """All values of a sign and exponent range against the block's largest magnitude at the borders of its scale."""
    from sharpinference_amd import ops
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    rows = []
    for top in (1.0, 1.7421875, 1.75, 1.7578125, 1.9921875):
        for power in (-130, -126, -118, -20, 0, 8, 9, 100, 127):
            t = torch.tensor([top * 2.0 ** power], dtype=torch.float64).bfloat16()
            v = torch.where(every.abs() <= t, every, torch.zeros_like(every))
            v = torch.cat([v, v.new_zeros(127 - v.numel() % 127)]).view(-1, 127)
            rows.append(torch.cat([v, t.expand(v.shape[0], 1)], 1))
    x = torch.cat(rows).to(DEV)
    _rows_check(x, ops.quantize_rows(x), x)
    _rows_check(x, ops.quantize_rows(x.float()), x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [128, 300])
def test_values_that_are_not_finite(K, dtype):
    from sharpinference_amd import ops
    x = _normal(_gen(K), 9, K).to(dtype)
    x[1, 3], x[2, 5], x[3, 7], x[4, :] = float("inf"), float("-inf"), float("nan"), float("nan")
    x[5, :] = 0
    x[6, K - 1] = torch.finfo(dtype).max
    x[7, 0] = float("-nan")
    q = ops.quantize_rows(x)
    _rows_check(x, q, x)
    assert q.codes.double()[1:5].isnan().sum() == 3 + K


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh", ("swish_clamp", 7.0)])
@pytest.mark.parametrize("M,K", [(1, 8), (7, 129), (65, 1403), (300, 512)])
def test_gated_rows_are_those_of_the_activation(M, K, act, dtype):
    from sharpinference_amd import ops
    x = _normal(_gen(M, K), M, 2 * K, scale=3.0).to(dtype)
    h = ops.gated_act(x, None, plain.code(act))
    _rows_check(x, ops.quantize_rows(x, plain.code(act)), h)


def _weight(g, *shape, gated=False, whole=False):
    from sharpinference_amd import ops
    w = _whole(g, *shape) if whole else _normal(g, *shape, scale=0.02)
    return w, ops.quantize_weight(w, gated)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape", [(2, 1), (32, 128), (34, 129), (500, 700), (3, 66, 300)])
def test_weights_keep_their_values(shape, gated):
    from sharpinference_amd import ops
    w, p = _weight(_gen(*shape), *shape, gated=gated)
    want = plain.rows(w.view(-1, shape[-1])).view(shape)
    assert torch.equal(p.values().double(), want)
    K = shape[-1]
    codes, e = plain.quantised(w.view(-1, K))
    again = ops.fp8_weight(codes[:, :K].float().to(F8).view(shape), (e + 127).to(torch.uint8).view(*shape[:-1], -1), gated)
    assert torch.equal(again.codes, p.codes) and torch.equal(again.scales, p.scales)
    if len(shape) == 3:
        assert torch.equal(p.select(1).values().double(), want[1])


LINEAR = [(1, 1, 1), (1, 16, 128), (2, 33, 129), (3, 5120, 512), (16, 70, 1000), (17, 100, 300), (32, 257, 511), (33, 64, 128), (64, 1030, 2000),
          (65, 1, 1), (65, 33, 130), (100, 300, 1028), (128, 256, 128), (129, 512, 384), (300, 70, 640), (513, 1040, 1536), (1000, 259, 2100)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", LINEAR)
def test_products(M, N, K, dtype):
    from sharpinference_amd import ops
    g = _gen(M, N, K)
    x = (_normal(g, M, K) * torch.exp(_normal(g, M, 1))).to(dtype)
    w, p = _weight(g, N, K)
    y = ops.linear_fp8(x, p)
    a, b = plain.rows(x), plain.rows(w)
    want = a @ b.T
    assert y.dtype == torch.bfloat16 and y.shape == (M, N)
    assert ((y.double() - want).abs() <= plain.cut(a, b) + plain.stored(want)).all()
    q = ops.quantize_rows(x)
    assert torch.equal(ops.linear_fp8(q, p), y)


@pytest.mark.parametrize("M", [1, 16, 40, 200])
def test_products_of_whole_numbers_are_exact(M):
    """Blocks of very different scales: sums that float holds exactly."""
    from sharpinference_amd import ops
    g = _gen(M)
    K, N = 520, 96
    x, w = _whole(g, M, K), _whole(g, N, K)
    x[:, 128:256] *= 2.0 ** 10
    w[:, 128:256] *= 2.0 ** -10
    w[:, 256:384] *= 64
    x[:, 256:384] /= 64
    want = x.double() @ w.double().T
    assert torch.equal(ops.linear_fp8(x, ops.quantize_weight(w)), want.to(torch.bfloat16))


@pytest.mark.parametrize("M", [4, 16, 60, 130])
def test_rows_that_are_not_finite_stay_apart(M):
    from sharpinference_amd import ops
    g = _gen(M)
    w, p = _weight(g, 200, 384)
    x = _normal(g, M, 384).bfloat16()
    clean = ops.linear_fp8(x, p)
    x[1, 3], x[M - 1, 200] = float("inf"), float("nan")
    y = ops.linear_fp8(x, p)
    keep = torch.ones(M, dtype=torch.bool, device=DEV)
    keep[[1, M - 1]] = False
    assert torch.equal(y[keep], clean[keep]) and y[~keep].isnan().all()


@pytest.mark.parametrize("M", [5, 16, 50, 200])
def test_rows_from_any_address(M):
    from sharpinference_amd import ops
    g = _gen(M)
    w, p = _weight(g, 100, 256)
    store = _normal(g, M * 256 + 3).bfloat16()
    x = store[3:].view(M, 256)
    assert x.data_ptr() % 16 and torch.equal(ops.linear_fp8(x, p), ops.linear_fp8(x.clone(), p))


def _picks(g, T, E, k, distinct=True):
    ids = torch.stack([torch.randperm(E, generator=g, device=DEV)[:k] if distinct else torch.randint(0, E, (k,), generator=g, device=DEV) for _ in range(T)])
    return ids.int().contiguous(), torch.rand(T, k, generator=g, device=DEV).contiguous() + 0.1


FEED = [(1, 128, 128), (1, 300, 70), (8, 512, 640), (16, 130, 33), (17, 256, 200), (40, 300, 1030), (64, 128, 257), (65, 128, 128), (100, 300, 70), (200, 640, 500), (600, 256, 390)]


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", ("swish_clamp", 7.0)])
@pytest.mark.parametrize("M,K,I", FEED)
def test_feed_forwards(M, K, I, act):
    from sharpinference_amd import ops
    g = _gen(M, K, I)
    x = _whole(g, M, K).bfloat16()
    w1, p1 = _weight(g, 2 * I, K, gated=True, whole=True)
    w1, p1 = w1 / 64, ops.quantize_weight(w1 / 64, True)
    w2, p2 = _weight(g, K + 3, I)
    y = ops.feed_forward_fp8(x, p1, p2, plain.code(act))
    want, bound = plain.feed_forward(x.double(), w1.double(), plain.rows(w2), act)
    assert ((y.double() - want).abs() <= bound + plain.stored(want)).all()
    assert torch.equal(ops.feed_forward_fp8(x.float(), p1, p2, plain.code(act)), y)
    assert torch.equal(ops.feed_forward_fp8(ops.quantize_rows(x), p1, p2, plain.code(act)), y)


EXPERTS = [(1, 1, 1, 128, 128, 128, False), (1, 4, 1, 256, 130, 100, True), (2, 8, 8, 128, 40, 300, False), (5, 100, 6, 300, 70, 257, False), (16, 16, 1, 256, 200, 128, True),
           (16, 5, 3, 130, 129, 64, False), (17, 16, 2, 128, 128, 256, True), (33, 64, 6, 256, 100, 130, False), (64, 8, 2, 300, 70, 96, True),
           (65, 4, 1, 128, 128, 128, False), (100, 28, 4, 256, 130, 200, True), (300, 8, 2, 300, 260, 140, False), (700, 3, 1, 256, 390, 300, True)]


def _layer(g, E, K, I, N, shared):
    from sharpinference_amd import ops
    n = E + (1 if shared else 0)
    w1 = _whole(g, n, 2 * I, K) / 64
    w2 = _normal(g, n, N, I, scale=0.02)
    return w1, w2, ops.quantize_weight(w1, True), ops.quantize_weight(w2)


def _layer_want(x, ids, wts, w1, w2, act, on_input, shared):
    T, k = ids.shape
    E = w1.shape[0] - (1 if shared else 0)
    want = torch.zeros(T, w2.shape[1], dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(want)
    for e in range(E + (1 if shared else 0)):
        a, b = w1[e].double(), plain.rows(w2[e])
        for j in range(k if e < E else 1):
            at = torch.nonzero(ids[:, j] == e).flatten() if e < E else torch.arange(T, device=DEV)
            if at.numel() == 0:
                continue
            s = wts[at, j] if e < E else None
            y, d = plain.feed_forward(x[at].double(), a, b, act, s if on_input else None)
            f = s[:, None].double() if s is not None and not on_input else 1.0
            want[at] += y * f
            bound[at] += d * f
    return want, bound


@pytest.mark.parametrize("on_input", [False, True])
@pytest.mark.parametrize("T,E,k,K,I,N,shared", EXPERTS)
def test_layers_of_experts(T, E, k, K, I, N, shared, on_input):
    from sharpinference_amd import ops
    g = _gen(T, E, k, K, I, N)
    x = _whole(g, T, K).bfloat16()
    w1, w2, p1, p2 = _layer(g, E, K, I, N, shared)
    ids, wts = _picks(g, T, E, k)
    y = ops.experts_fp8(x, ids, wts, p1, p2, score_on_input=on_input, shared=shared)
    want, bound = _layer_want(x, ids, wts, w1, w2, "silu", on_input, shared)
    assert ((y.double() - want).abs() <= bound + 2 ** -20 * want.abs() + plain.stored(want)).all()
    for _ in range(3):
        assert torch.equal(ops.experts_fp8(x, ids, wts, p1, p2, score_on_input=on_input, shared=shared), y)


@pytest.mark.parametrize("T,shared", [(6, False), (6, True), (40, True), (90, False), (90, True)])
def test_a_token_that_picks_an_expert_twice_and_one_that_is_not_there(T, shared):
    from sharpinference_amd import ops
    g = _gen(T)
    E, k, K, I, N = 5, 4, 128, 96, 70
    x = _whole(g, T, K).bfloat16()
    w1, w2, p1, p2 = _layer(g, E, K, I, N, shared)
    ids, wts = _picks(g, T, E, k, distinct=False)
    ids[0] = 3
    ids[1] = torch.tensor([E, E + 2, 1, 1], device=DEV)
    ids[2] = E
    for on_input in (False, True):
        y = ops.experts_fp8(x, ids, wts, p1, p2, score_on_input=on_input, shared=shared)
        want, bound = _layer_want(x, ids, wts, w1, w2, "silu", on_input, shared)
        assert ((y.double() - want).abs() <= bound + 2 ** -20 * want.abs() + plain.stored(want)).all()


def test_nothing_to_do():
    from sharpinference_amd import ops
    g = _gen(1)
    w1, w2, p1, p2 = _layer(g, 2, 128, 64, 96, False)
    x = torch.empty(0, 128, dtype=torch.bfloat16, device=DEV)
    assert ops.quantize_rows(x).shape == (0, 128)
    assert ops.linear_fp8(x, ops.quantize_weight(_normal(g, 5, 128))).shape == (0, 5)
    assert ops.feed_forward_fp8(x, p1.select(0), p2.select(0)).shape == (0, 96)
    ids, wts = torch.empty(0, 2, dtype=torch.int32, device=DEV), torch.empty(0, 2, device=DEV)
    assert ops.experts_fp8(x, ids, wts, p1, p2).shape == (0, 96)


def _operators(g):
    """name -> (inputs that change, call on them) of every operator, for few and many rows."""
    from sharpinference_amd import ops
    _, lin = _weight(g, 200, 384)
    w1, w2, p1, p2 = _layer(g, 8, 384, 160, 200, True)
    out = {}
    for M in (1, 3, 16, 40, 130):
        x = _normal(g, M, 384).bfloat16()
        ids, wts = _picks(g, M, 8, 2)
        out[f"rows {M}"] = ([x], lambda x: ops.quantize_rows(x).values())
        out[f"gated rows {M}"] = ([_normal(g, M, 768)], lambda x: ops.quantize_rows(x, ops.ACT_SILU).values())
        out[f"linear {M}"] = ([x], lambda x: ops.linear_fp8(x, lin))
        out[f"feed forward {M}"] = ([x], lambda x: ops.feed_forward_fp8(x, p1.select(8), p2.select(8)))
        out[f"experts {M}"] = ([x, ids, wts], lambda x, ids, wts: ops.experts_fp8(x, ids, wts, p1, p2, shared=True))
    return out


def test_captured_calls_replay_on_new_inputs():
    g = _gen(5)
    for name, (inputs, call) in _operators(g).items():
        static = [t.clone() for t in inputs]
        call(*static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(*static)
        for turn in range(4):
            for s, t in zip(static, inputs):
                s.copy_(t.flip(0) if turn % 2 else t)
            want = call(*[t.clone() for t in static])          # (eager work between the replays)
            torch.cuda.synchronize()
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), (name, turn)


def test_two_captured_layers_replayed_side_by_side():
    """Graphs of one operator on two streams share nothing."""
    g = _gen(6)
    (inputs, call), graphs = _operators(g)["experts 3"], []
    want = call(*inputs)
    for _ in range(2):
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call(*inputs)
        graphs.append((stream, graph, out))
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, graph, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, _, out in graphs)


def test_calls_on_streams_of_their_own():
    g = _gen(7)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for name, (inputs, call) in _operators(g).items():
        want, got = call(*inputs), []
        torch.cuda.synchronize()
        for _ in range(3):
            for s in streams:
                with torch.cuda.stream(s):
                    got.append(call(*inputs))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in got), name


def test_a_run_of_them_as_a_layer_uses_them():
    """Quantised once, multiplied twice: a projection and a layer of experts over the same rows, then the projection of their sum."""
    from sharpinference_amd import ops
    g = _gen(8)
    _, lin = _weight(g, 384, 384)
    _, _, p1, p2 = _layer(g, 4, 384, 160, 384, True)
    for M in (2, 50, 300):
        x = _normal(g, M, 384).bfloat16()
        ids, wts = _picks(g, M, 4, 2)
        q = ops.quantize_rows(x)
        a, b = ops.linear_fp8(q, lin), ops.experts_fp8(q, ids, wts, p1, p2, shared=True)
        assert torch.equal(a, ops.linear_fp8(x, lin)) and torch.equal(b, ops.experts_fp8(x, ids, wts, p1, p2, shared=True))
        y = ops.linear_fp8(a + b, lin)
        s, w = plain.rows(a + b), lin.values().double()
        want = s @ w.T
        assert ((y.double() - want).abs() <= plain.cut(s, w) + plain.stored(want)).all()


def test_columns_behind_the_last_and_rows_beside_stay_as_they_are():
    """A result's neighbours in memory are not written (odd sizes: stores of whole runs would pass the end)."""
    from sharpinference_amd import ops
    from sharpinference_amd.ops import fp8
    g = _gen(9)
    for M in (1, 5, 16, 33, 70, 200):
        for N in (1, 33, 100, 257):
            _, w = _weight(g, N, 256)
            x = _normal(g, M, 256).bfloat16()
            want = ops.linear_fp8(x, w)
            q = ops.quantize_rows(x)
            room = torch.full((M * N + 256,), 7.0, dtype=torch.bfloat16, device=DEV)
            out = room[64:64 + M * N]
            if M <= 64:
                ops._run("sharpi_fp8_few", q.codes.data_ptr(), q.scales.data_ptr(), 2, w.codes.data_ptr(), w.scales.data_ptr(), w.stored_rows, out.data_ptr(),
                         M, N, 256, 1, ops._stream())
            else:
                ops._run("sharpi_fp8_tiles", q.codes.data_ptr(), q.scales.data_ptr(), M, w.codes.data_ptr(), w.scales.data_ptr(), w.stored_rows,
                         out.data_ptr(), 1, M, N, 256, None, None, 1, 0, 128, 2, 1, ops._stream())
            torch.cuda.synchronize()
            assert torch.equal(out.view(M, N), want) or ((out.view(M, N).double() - want.double()).abs() <= 2 * plain.stored(want.double()) + 1e-3).all()
            assert (room[:64] == 7).all() and (room[64 + M * N:] == 7).all()
    assert fp8.FP8_FEW_ROWS == 64


@pytest.mark.parametrize("M,N,K", [(100, 96, 1100), (70, 513, 2048), (300, 100, 520)])
@pytest.mark.parametrize("tile", [(64, 2, 1), (64, 2, 3), (128, 2, 2), (192, 1, 1), (192, 1, 4), (192, 2, 2), (256, 1, 3), (256, 2, 1), (256, 2, 4)])
def test_products_in_every_kind_of_tile(monkeypatch, M, N, K, tile):
    """Every height, width and number of shares, whatever the rule would choose."""
    from sharpinference_amd import ops
    from sharpinference_amd.ops import fp8
    g = _gen(M, N, K)
    x = (_normal(g, M, K) * torch.exp(_normal(g, M, 1))).bfloat16()
    w, p = _weight(g, N, K)
    monkeypatch.setattr(fp8, "tile_fp8", lambda *a: tile)
    y = ops.linear_fp8(x, p)
    a, b = plain.rows(x), plain.rows(w)
    want = a @ b.T
    assert ((y.double() - want).abs() <= plain.cut(a, b) + plain.stored(want)).all()


@pytest.mark.parametrize("height", [64, 128, 192, 256])
@pytest.mark.parametrize("T,E,k,shared", [(90, 4, 2, True), (700, 3, 1, False), (500, 2, 2, True)])
def test_layers_in_every_height_of_tile(monkeypatch, T, E, k, shared, height):
    from sharpinference_amd import ops
    from sharpinference_amd.ops import fp8
    g = _gen(T, E, k)
    x = _whole(g, T, 256).bfloat16()
    w1, w2, p1, p2 = _layer(g, E, 256, 200, 140, shared)
    ids, wts = _picks(g, T, E, k)
    monkeypatch.setattr(fp8, "grouped_tile_fp8", lambda *a: height)
    y = ops.experts_fp8(x, ids, wts, p1, p2, shared=shared)
    want, bound = _layer_want(x, ids, wts, w1, w2, "silu", False, shared)
    assert ((y.double() - want).abs() <= bound + 2 ** -20 * want.abs() + plain.stored(want)).all()


def test_refused_on_the_gpu():
    from sharpinference_amd import ops
    g = _gen(3)
    _, w = _weight(g, 64, 128)
    x = _normal(g, 4, 256).bfloat16()
    for bad in (x, x[:, ::2], x[:, :128].half(), x[0, :128], ops.quantize_rows(x)):
        with pytest.raises(ops.KernelError):
            ops.linear_fp8(bad, w)
    _, _, p1, p2 = _layer(g, 3, 128, 64, 96, False)
    x, (ids, wts) = _normal(g, 4, 128).bfloat16(), _picks(g, 4, 3, 2)
    for a, b in ((ids.long(), wts), (ids, wts.double()), (ids[:3], wts[:3]), (ids, wts[:, :1]), (ids.cpu(), wts), (ids.t().contiguous().t(), wts)):
        with pytest.raises(ops.KernelError):
            ops.experts_fp8(x, a, b, p1, p2)
    with pytest.raises(ops.KernelError, match="not known"):
        ops.experts_fp8(x, ids, wts, p1, p2, act=9)
    with pytest.raises(ops.KernelError):
        ops.feed_forward_fp8(x, p1.select(0), p2.select(0), act=(ops.ACT_SWISH_CLAMP, -1.0))
    with pytest.raises(ops.KernelError):
        ops.quantize_rows(_normal(g, 3, 5), ops.ACT_SILU)
