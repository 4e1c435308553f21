"""adapter_linear(): against 64 bits over requests of every size, ids without an adapter, epilogues and forms of the launch; refusals.

Tolerance, per element. Products of fp16 are exact in fp32; a step of the tensor core adds 16 of them to the accumulator, off by at
most 2^-23 of the sum of magnitudes so far, with 17 more such roundings inside the steps: (K / 16 + 17) 2^-23 sum |x w|. (On the CUDA
cores a sum of r or K / 64 terms a lane, then of 32 lanes, stays below that.) h = scale (x down') is off likewise and rounded to fp16: 2^-11
of it, or half of fp16's smallest step, 2^-25; |h|'s error times |up| adds up over the rank. GELU's slope is below 1.13 (its erf 7.1e-7),
silu's below 1.1 (its exponential and reciprocal 2^-20 of the value). gamma scales all that; fp32 roundings on the way, 2^-22 of the
magnitudes; the result is rounded to fp16: 2^-11 of it, or 2^-25."""
import math

import pytest
import torch

from fastbb_b200 import _lib
from fastbb_b200.adapters import Adapters, adapter_linear


def reference(x, w, slots, ids, bounds, b=None, act=None, res=None, gamma=None):
    """(y, room) in 64 bits; bounds: first row of each request and the end of the last."""
    K, N = x.shape[-1], w.shape[0]
    x = x.reshape(-1, K).double()
    step = lambda k: (k / 16 + 17) * 2.0 ** -23  # noqa: E731
    y, room = x @ w.double().t(), step(K) * (x.abs() @ w.double().abs().t())
    for s, a in enumerate(ids):
        rows = slice(min(max(bounds[s], 0), x.shape[0]), min(max(bounds[s + 1], 0), x.shape[0]))
        if not 0 <= a < slots.count or rows.stop <= rows.start:
            continue
        down, up, scale = slots.down[a].double(), slots.up[a].double(), float(slots.scale[a])
        h = scale * (x[rows] @ down.t())
        dh = abs(scale) * step(K) * (x[rows].abs() @ down.abs().t()) + h.abs() * 2.0 ** -11 + 2.0 ** -25
        y[rows] += h @ up.t()
        room[rows] += dh @ up.abs().t() + step(K + slots.rank) * ((h.abs() + dh) @ up.abs().t())
    if b is not None:
        y = y + b.double()
    room = room + y.abs() * 2.0 ** -22
    if act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
        room = 1.13 * room + 7.2e-7
    elif act == "swiglu":
        x1, x2 = y.chunk(2, -1)
        r1, r2 = room.chunk(2, -1)
        y = x1 * torch.sigmoid(x1) * x2
        room = 1.1 * r1 * (x2.abs() + r2) + (x1 * torch.sigmoid(x1)).abs() * r2 + y.abs() * 2.0 ** -20
    if res is not None:
        f = 1.0 if gamma is None else gamma.double()
        y = res.reshape(y.shape).double() + f * y
        room = room * (f if gamma is None else f.abs()) + (y.abs() + res.reshape(y.shape).double().abs()) * 2.0 ** -22
    return y, room + y.abs() * 2.0 ** -11 + 2.0 ** -25


def check(got, *args, **kw):
    want, room = reference(*args, **kw)
    over = (got.reshape(want.shape).double() - want).abs() - room
    assert bool((over <= 0).all()), f"{int((~(over <= 0)).sum())} of {over.numel()} off, worst by {float(over.max()):.3g}, room there {float(room.flatten()[over.argmax()]):.3g}"


def make(M, K, N, r, L, g):
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).half()  # noqa: E731
    slots = Adapters(rnd(L, r, K, std=K ** -0.5), rnd(L, N, r, std=0.1), torch.rand(L, generator=g, device="cuda") + 0.5)
    return rnd(M, K), rnd(N, K, std=K ** -0.5), slots, rnd(N, std=0.3)


def vector(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "gelu", "swiglu", "res"])
@pytest.mark.parametrize("S,each,K,N,r,L", [
    (1, 1, 8, 16, 8, 1), (1, 1, 1024, 1024, 16, 3), (5, 1, 72, 144, 24, 2), (64, 1, 384, 384, 16, 40), (130, 1, 256, 512, 64, 7), (33, 7, 128, 272, 32, 5),
    (2, 9, 768, 768, 8, 2), (3, 37, 200, 336, 40, 3), (8, 257, 384, 1152, 16, 6), (40, 32, 96, 256, 128, 9), (4, 128, 512, 512, 16, 4), (1, 3000, 256, 1024, 32, 1),
    (2, 1370, 1536, 1536, 64, 3), (13, 256, 128, 1536, 104, 20), (300, 9, 64, 1024, 8, 50)])
def test_matches_64_bits(S, each, K, N, r, L, act):
    g = torch.Generator("cuda").manual_seed(S * 1000 + each + r)
    x, w, slots, b = make(S * each, K, N, r, L, g)
    ids = [(s * 7 + 3) % (L + 1) - 1 for s in range(S)]
    kw = {"b": b, "act": None if act == "res" else act}
    if act == "res":
        kw["res"], kw["gamma"] = torch.randn(S, each, N, generator=g, device="cuda").half(), torch.randn(N, generator=g, device="cuda").half()
    out = adapter_linear(x.view(S, each, K), w, slots, vector(ids), **kw)
    assert out.shape == (S, each, N // 2 if act == "swiglu" else N)
    check(out, x, w, slots, ids, [s * each for s in range(S + 1)], **kw)
    assert torch.equal(out, adapter_linear(x.view(S, each, K), w, slots, vector(ids), **kw))
    assert _lib.device_status() == (0, 0, 0, 0)


RAGGED = [[0, 1], [0, 0, 5, 5, 5, 6, 300], [3, 40, 41, 90], [0, 127, 128, 129, 255, 256, 257, 600, 600], [0, 1, 2, 3, 4, 5, 6, 7, 2000], [7, 7, 7], [0, 2500, 2501, 2502, 4100]]


@pytest.mark.gpu
@pytest.mark.parametrize("bounds", RAGGED)
@pytest.mark.parametrize("behind", [0, 1, 130])
def test_requests_of_any_size_one_behind_another(bounds, behind):
    g = torch.Generator("cuda").manual_seed(len(bounds) + behind)
    M, S = bounds[-1] + behind, len(bounds) - 1
    x, w, slots, b = make(M, 192, 640, 16, 4, g)
    ids = [(s * 5 + 1) % 6 - 1 for s in range(S)]  # -1 and 4 are no adapter
    out = adapter_linear(x, w, slots, vector(ids), vector(bounds), b=b)
    check(out, x, w, slots, ids, bounds, b=b)
    res = torch.randn(M, 640, generator=g, device="cuda").half()
    want = adapter_linear(x, w, slots, vector(ids), vector(bounds), b=b, res=res)
    assert adapter_linear(x, w, slots, vector(ids), vector(bounds), b=b, res=res, out=res) is res and torch.equal(res, want)  # in place on the residual


@pytest.mark.gpu
def test_many_requests_of_few_and_of_many_rows():
    g = torch.Generator("cuda").manual_seed(3)
    counts = [0, 1, 2, 3, 5, 8, 13, 21, 34, 55, 89, 144, 233, 377, 610, 0, 0, 1, 1, 1] * 3
    bounds = [0]
    for c in counts:
        bounds.append(bounds[-1] + c)
    ids = [(s * 3) % 11 - 1 for s in range(len(counts))]
    x, w, slots, b = make(bounds[-1], 256, 1024, 16, 10, g)
    check(adapter_linear(x, w, slots, vector(ids), vector(bounds), b=b, act="gelu"), x, w, slots, ids, bounds, b=b, act="gelu")


def _bounds(counts, first=0):
    at = [first]
    for c in counts:
        at.append(at[-1] + c)
    return at


CROWDS = {
    "single rows": _bounds([1] * 300),                                                      # up to 128 requests in a tile of 128 rows, 256 in one of 256
    "pairs and gaps": _bounds([2, 0, 1, 0, 3] * 40, first=5),
    "empty ones between": _bounds([40] + [0] * 70 + [30] + [0] * 33 + [1] * 40 + [0] * 32 + [300]),  # whole rounds of 32 look-ups without a row
    "growing": _bounds([i * i // 16 for i in range(48)]),
    "forty rows each": _bounds([40] * 13)}


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["r", "s64", "s128", "p256"])
@pytest.mark.parametrize("crowd", CROWDS)
@pytest.mark.parametrize("rank,act", [(8, "gelu"), (24, "swiglu"), (40, "res"), (64, None), (128, "swiglu")])
def test_every_form_with_few_and_many_requests_in_a_tile(form, crowd, rank, act, monkeypatch):
    """The form is forced, so that each one has all of these, whatever the rule that picks one."""
    monkeypatch.setenv("FBB_ADAPTER_FORM", form)
    g = torch.Generator("cuda").manual_seed(rank + len(crowd))
    bounds, (K, N, L) = CROWDS[crowd], (200, 656, 7)
    M, S = bounds[-1] + 3, len(bounds) - 1
    x, w, slots, b = make(M, K, N, rank, L, g)
    ids = [(s * 5 + 2) % (L + 2) - 1 for s in range(S)]  # -1 and L are no adapter
    kw = {"b": b, "act": None if act == "res" else act}
    if act == "res":
        kw["res"], kw["gamma"] = torch.randn(M, N, generator=g, device="cuda").half(), torch.randn(N, generator=g, device="cuda").half()
    need = _lib.load().fbb_adapter_linear_workspace_bytes(M, N, K, _lib.EPI_SWIGLU if act == "swiglu" else _lib.EPI_NONE, rank, S)
    assert need == (M * N * 4 if form == "r" else M * rank * 2 + (M + 255) // 256 * 32)  # what the rows form and the blocks form keep
    out = adapter_linear(x, w, slots, vector(ids), vector(bounds), **kw)
    check(out, x, w, slots, ids, bounds, **kw)
    assert torch.equal(out, adapter_linear(x, w, slots, vector(ids), vector(bounds), **kw))
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["r", "s64", "s128", "p256"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_infinite_values_stay_in_their_rows_in_every_form(form, bad, monkeypatch):
    monkeypatch.setenv("FBB_ADAPTER_FORM", form)
    g = torch.Generator("cuda").manual_seed(6)
    bounds = CROWDS["pairs and gaps"]
    M, S, K, N = bounds[-1], len(bounds) - 1, 128, 320
    x, w, slots, b = make(M, K, N, 16, 3, g)
    ids = [s % 3 for s in range(S)]
    clean = adapter_linear(x, w, slots, vector(ids), vector(bounds), b=b)
    hit = torch.zeros(M, dtype=torch.bool, device="cuda")
    for s in range(S):
        hit[bounds[s]:bounds[s + 1]] = ids[s] == 1
    for matrix in (slots.up, slots.down):
        kept = matrix[1].clone()
        matrix[1] = bad
        out = adapter_linear(x, w, slots, vector(ids), vector(bounds), b=b)
        assert torch.equal(out[~hit], clean[~hit]) and not bool(out[hit].isfinite().any())
        matrix[1] = kept


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["r", "s64", "s128", "p256"])
@pytest.mark.parametrize("crowd", CROWDS)
@pytest.mark.parametrize("rank,act", [(8, "gelu"), (40, "res"), (72, None), (128, "swiglu")])
def test_first_products_beyond_fp16(form, crowd, rank, act, monkeypatch):
    """Rows of h up to about 3e7 beside rows that fp16 holds, in one request and in others of the tile. Rows beyond fp16 are held times 2^-15: fp16's
    smallest step is 2^-10 of theirs, half of that on top of the tolerance (2^-25 of it is there already)."""
    monkeypatch.setenv("FBB_ADAPTER_FORM", form)
    g = torch.Generator("cuda").manual_seed(rank + len(crowd))
    bounds, (K, N, L) = CROWDS[crowd], (200, 656, 3)
    M, S = bounds[-1], len(bounds) - 1
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (rnd(M, K) * torch.tensor([1.0, 10.0, 1000.0, 10000.0], device="cuda")[torch.randint(0, 4, (M, 1), generator=g, device="cuda")]).clamp(-60000, 60000).half()
    scales = [0.7, 100.0, 3.0] if act != "swiglu" else [0.7, 10.0, 3.0]
    slots = Adapters(rnd(L, rank, K).half(), (rnd(L, N, rank) * (2e-5 if act != "swiglu" else 2e-6)).half(), torch.tensor(scales, device="cuda"))
    w, b, ids = (rnd(N, K) * 1e-4).half(), rnd(N).half(), [s % 4 for s in range(S)]  # 3 is no adapter
    kw = {"b": b, "act": None if act == "res" else act}
    if act == "res":
        kw["res"], kw["gamma"] = rnd(M, N).half(), rnd(N).half()
    want, room = reference(x, w, slots, ids, bounds, **kw)
    most = max(float((slots.scale[a] * (x[bounds[s]:bounds[s + 1]].float() @ slots.down[a].float().t())).abs().max()) for s, a in enumerate(ids)
               if a < L and bounds[s] < bounds[s + 1])
    assert most > 1e6 and float(want.abs().max()) < 6e4
    small = 2.0 ** -11 * float(slots.up.float().abs().sum(-1).max())
    if act == "swiglu":
        y = x.double() @ w.double().t() + b.double()
        small *= 1.2 * float(want.abs().max() ** 0.5 + y.abs().max() + 60)  # (times the other half's values)
    elif act == "res":
        small = small * kw["gamma"].double().abs()
    else:
        small *= 1.13
    out = adapter_linear(x, w, slots, vector(ids), vector(bounds), **kw)
    over = (out.double() - want).abs() - room - small
    assert bool((over <= 0).all()), f"{int((~(over <= 0)).sum())} of {over.numel()} off, worst by {float(over.max()):.3g}"
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("bounds,K,N,r", [(_bounds([40] * 64), 1024, 1024, 8), (_bounds([6145 * i * i // 85344 for i in range(64)]), 1024, 1024, 32),
                                          (_bounds([1] * 2000), 384, 1536, 16)])
def test_batches_of_many_requests_in_the_form_that_the_rule_picks(bounds, K, N, r):
    g = torch.Generator("cuda").manual_seed(K + r)
    S = len(bounds) - 1
    x, w, slots, b = make(bounds[-1], K, N, r, 48, g)
    ids = [-1 if s % 5 == 4 else s * 7 % 48 for s in range(S)]
    check(adapter_linear(x, w, slots, vector(ids), vector(bounds), b=b), x, w, slots, ids, bounds, b=b)
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.gpu
def test_without_any_adapter_it_is_the_linear_layer():
    from fastbb_b200.gemm import linear
    g = torch.Generator("cuda").manual_seed(4)
    for S, each in ((6, 300), (50, 1)):
        x, w, slots, b = make(S * each, 320, 512, 16, 2, g)
        y = linear(x, w, b, act="gelu").float()
        out = adapter_linear(x.view(S, each, 320), w, slots, vector([-1] * S), b=b, act="gelu").view(-1, 512).float()
        # the same fp16 operands and fp32 sums, in another order at most: one rounding to fp16 apart
        assert float((out - y).abs().max()) <= 2.0 ** -10 * float(y.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("M,N,bounds", [(300, 256, [0, 100, 130, 300]), (3000, 1024, [0, 1000, 1033, 3000]), (40, 512, [0, 1, 2, 40])])
def test_infinite_values_stay_in_their_rows(M, N, bounds, bad):
    """A request's NaN and infinities, in its rows of x or in its adapter, reach only its rows, though tiles hold several requests."""
    g = torch.Generator("cuda").manual_seed(5)
    ids = [0, 1, 0]
    x, w, slots, b = make(M, 128, N, 16, 2, g)
    rows = slice(bounds[1], bounds[2])
    clean = adapter_linear(x, w, slots, vector(ids), vector(bounds), b=b)

    def others_are_clean():
        out = adapter_linear(x, w, slots, vector(ids), vector(bounds), b=b)
        assert torch.equal(out[:rows.start], clean[:rows.start]) and torch.equal(out[rows.stop:], clean[rows.stop:])
        return out[rows]

    kept = x[rows, 5].clone()
    x[rows, 5] = bad
    assert not bool(others_are_clean().isfinite().any())
    x[rows, 5] = kept
    for matrix in (slots.up, slots.down):
        kept_matrix = matrix[1].clone()
        matrix[1] = bad
        assert not bool(others_are_clean().isfinite().any())
        matrix[1] = kept_matrix
    slots.scale[1] = bad
    assert not bool(others_are_clean().isfinite().any())


@pytest.mark.gpu
def test_row_strides_and_a_weight_view():
    g = torch.Generator("cuda").manual_seed(6)
    x, w, slots, b = make(450, 128, 512, 32, 3, g)
    wide_x, wide_w = torch.randn(450, 200, generator=g, device="cuda").half(), torch.randn(512, 136, generator=g, device="cuda").half()
    wide_x[:, 8:136], wide_w[:, :128] = x, w
    res = torch.randn(450, 1024, generator=g, device="cuda").half()[:, 512:]
    ids, bounds = [2, 0], [0, 200, 450]
    out = adapter_linear(wide_x[:, 8:136], wide_w[:, :128], slots, vector(ids), vector(bounds), b=b, res=res)
    check(out, x, w, slots, ids, bounds, b=b, res=res)


@pytest.mark.gpu
def test_other_stream_and_graphs_that_live_side_by_side():
    g = torch.Generator("cuda").manual_seed(7)
    sets = []
    for S, each in ((40, 1), (3, 70), (7, 500)):
        x, w, slots, b = make(S * each, 256, 768, 16, 5, g)
        sets.append((x.view(S, each, 256), w, slots, vector([s % 5 for s in range(S)]), None, b))
    want = [adapter_linear(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [adapter_linear(*s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, adapter_linear(*s)))
    for s in sets:
        s[3].copy_(vector([(i + 2) % 6 - 1 for i in range(s[3].numel())]))  # a captured call reads the ids of its replay
    again = [adapter_linear(*s) for s in sets]
    for graph, _ in graphs + graphs:
        graph.replay()
    for o, w_, (_, c), a in zip(other, want, graphs, again):
        assert torch.equal(o, w_) and torch.equal(c, a) and not torch.equal(a, w_)


@pytest.mark.gpu
def test_a_call_behind_calls_that_make_its_inputs():
    """The second launch starts under the first: inputs written right before the call, and outputs read right behind it, are whole."""
    from fastbb_b200.gemm import linear
    g = torch.Generator("cuda").manual_seed(8)
    x, w, slots, b = make(2000, 512, 512, 16, 3, g)
    w0 = torch.randn(512, 512, generator=g, device="cuda").half() * 0.04
    ids, bounds = vector([0, 2, 1]), vector([0, 700, 701, 2000])
    first = linear(x, w0)
    torch.cuda.synchronize()
    y = adapter_linear(first, w, slots, ids, bounds, b=b)
    torch.cuda.synchronize()
    want = linear(y, w0, act="gelu")
    torch.cuda.synchronize()
    for _ in range(20):
        assert torch.equal(linear(adapter_linear(linear(x, w0), w, slots, ids, bounds, b=b), w0, act="gelu"), want)


@pytest.mark.gpu
def test_empty_calls():
    g = torch.Generator("cuda").manual_seed(9)
    x, w, slots, b = make(4, 64, 128, 8, 2, g)
    assert adapter_linear(x[:0], w, slots, vector([0]), vector([0, 0]), b=b).shape == (0, 128)
    assert adapter_linear(x[:0].view(2, 0, 64), w, slots, vector([0, 1]), b=b).shape == (2, 0, 128)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    g = torch.Generator("cuda").manual_seed(10)
    x, w, slots, b = make(12, 64, 128, 8, 2, g)
    x3, ids = x.view(3, 4, 64), vector([0, 1, -1])
    for call in (
            lambda: adapter_linear(x3, w, slots, vector([0, 1])), lambda: adapter_linear(x, w, slots, ids), lambda: adapter_linear(x3, w, slots, ids.long()),
            lambda: adapter_linear(x3, w, slots, ids.cpu()), lambda: adapter_linear(x, w, slots, ids, vector([0, 4, 12])),
            lambda: adapter_linear(x, w, slots, ids, vector([0, 4, 8, 12]).long()), lambda: adapter_linear(x3.float(), w, slots, ids),
            lambda: adapter_linear(x3, w[:, :56], slots, ids), lambda: adapter_linear(x3, w[:120], slots, ids), lambda: adapter_linear(x3, w, slots, ids, act="relu"),
            lambda: adapter_linear(x3, w, slots, ids, b=b[:5]), lambda: adapter_linear(x3, w, slots, ids, gamma=b),
            lambda: adapter_linear(x3, w, slots, ids, res=torch.zeros(12, 128, device="cuda").half()),
            lambda: adapter_linear(x3, w, slots, ids, out=torch.zeros(3, 4, 128, device="cuda")),
            lambda: adapter_linear(x[:, :64], torch.cat((w, w))[:64], Adapters(slots.down, slots.up[:, :64].contiguous()), ids, vector([0, 4, 8, 12]), out=x),
            lambda: Adapters(slots.down, slots.up[:1]), lambda: Adapters(slots.down.float(), slots.up), lambda: Adapters(slots.down[:, :4], slots.up[..., :4]),
            lambda: Adapters(slots.down, slots.up.transpose(1, 2).contiguous().transpose(1, 2)), lambda: Adapters(slots.down, slots.up, slots.scale.half()),
            lambda: Adapters(slots.down, slots.up, slots.scale[:1]), lambda: Adapters(slots.down[:0], slots.up[:0])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_lib.FastbbError):
        adapter_linear(x3, w, slots, ids, act="swiglu", res=torch.zeros(3, 4, 64, device="cuda").half())


@pytest.mark.gpu
def test_outputs_over_any_input_are_refused():
    """out shares its first bytes, or its last, with one input at a time; right behind it or ahead of it the call is taken."""
    g = torch.Generator("cuda").manual_seed(11)
    x, w, slots, b = make(16, 64, 128, 8, 2, g)
    ids, bounds, res, gamma = vector([0, 1, -1]), vector([0, 4, 12, 16]), torch.zeros(16, 128, device="cuda").half(), b.clone()
    size = 2 * 16 * 128
    store = torch.zeros(1 << 17, dtype=torch.uint8, device="cuda")
    parts = dict(x=x, w=w, b=b, gamma=gamma, down=slots.down, up=slots.up, scale=slots.scale, ids=ids, offsets=bounds, res=res)
    for name, t in parts.items():
        n, base = t.numel() * t.element_size(), 1 << 16
        for clear, shared in ((base + (n + 15) // 16 * 16, base + (n + 15) // 16 * 16 - 16), (base - size, base - size + 16)):
            view = store[base:base + n].view(t.dtype).view(t.shape)
            view.copy_(t)
            use = {**parts, name: view}
            call = lambda lo: adapter_linear(use["x"], use["w"], Adapters(use["down"], use["up"], use["scale"]), use["ids"], use["offsets"], b=use["b"],  # noqa: E731, B023
                                             res=use["res"], gamma=use["gamma"], out=store[lo:lo + size].view(torch.float16).view(16, 128))
            held = store.clone()
            with pytest.raises(ValueError, match="shares no memory"):
                call(shared)
            assert torch.equal(store, held)
            call(clear)


# ------------------------------------------------------------------------------------------------------------------ CPU
def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="no CPU path"):
        Adapters(torch.zeros(1, 8, 64).half(), torch.zeros(1, 128, 8).half())


def test_entry_point_refusals():
    lib, A = _lib.load(), 0x7F0000000000

    def call(a=A, w=A, c=A + (1 << 30), res=None, gamma=None, M=8, N=64, K=32, lda=32, ldw=32, ldc=64, ldr=64, epi=0, down=A, up=A, scale=A, L=2, r=16, ids=A,
             offsets=None, S=2, ws=A, bytes_=0):
        return lib.fbb_adapter_linear_f16(a, w, c, None, res, gamma, M, N, K, lda, ldw, ldc, ldr, epi, down, up, scale, L, r, ids, offsets, S, ws, bytes_, None)

    assert call(a=None) == call(w=None) == call(c=None) == call(down=None) == call(up=None) == call(scale=None) == call(ids=None) == -1
    assert call(K=12) == call(N=12) == call(lda=24) == call(ldw=24) == call(ldc=56) == call(res=A, ldr=8) == call(M=-1) == -2
    assert call(r=0) == call(r=12) == call(r=136) == call(L=0) == call(L=1 << 30) == call(S=0) == call(S=3) == call(c=A) == -2
    assert call(epi=2, res=A) == call(epi=2, N=72) == -2 and call(epi=3) == -4
    assert call(a=A + 8) == call(ws=A + 128) == call(up=A + 2) == call(ldc=68) == -3
    assert call(bytes_=64) == -2 and b"workspace" in lib.fbb_last_error()
    assert call(M=0, a=None) == 0
    assert lib.fbb_adapter_linear_workspace_bytes(0, 64, 64, 0, 8, 1) == 0


def test_more_rows_of_either_matrix_than_31_bits_count_are_refused():
    """(The workspace is the next thing that is refused: nothing is read or launched.)"""
    lib, A = _lib.load(), 0x7F0000000000

    def call(L, N, r):
        rc = lib.fbb_adapter_linear_f16(A, A, A + (1 << 30), None, None, None, 8, N, 32, 32, 32, N, 0, 0, A, A, A, L, r, A, None, 2, A, 0, None)
        return rc, b"2^31" in lib.fbb_last_error()

    assert call(1 << 24, 8, 128) == (-2, True) and call(1 << 28, 8, 8) == (-2, True) and call(1 << 20, 1 << 14, 8) == (-2, True)
    assert call((1 << 24) - 1, 8, 128)[1] is False


def test_the_record_form_refuses_what_the_other_does():
    """Every field is where the entry point looks for it: broken alone, it is the one that is named."""
    lib, A = _lib.load(), 0x7F0000000000
    good = dict(a=A, w=A, c=A + (1 << 30), b=A, res=A, gamma=A, down=A, up=A, scale=A, ids=A, offsets=A, ws=A, stream=0, M=8, lda=32, ldw=32, ldc=64, ldr=64,
                bytes_=0, N=64, K=32, epi=0, L=2, r=16, S=3)

    def call(**kw):
        return lib.fbb_adapter_linear_f16_from(_lib.AdapterLinearArgs.pack(*{**good, **kw}.values()))

    assert lib.fbb_adapter_linear_f16_from(None) == call(a=0) == call(w=0) == call(c=0) == call(down=0) == call(up=0) == call(scale=0) == call(ids=0) == -1
    assert call(offsets=0) == call(M=-1) == call(K=12) == call(N=12) == call(lda=24) == call(ldw=24) == call(ldc=56) == call(ldr=8) == call(c=A) == -2
    assert call(r=12) == call(L=0) == call(S=0) == call(epi=2) == -2 and call(epi=3) == -4 and call(epi=2, res=0) == -2
    assert call(res=A + 8) == call(up=A + 8) == call(down=A + 8) == call(ws=A + 128) == -3
    assert call(bytes_=64) == -2 and b"workspace of 64 bytes" in lib.fbb_last_error() and call(M=0, a=0) == 0
