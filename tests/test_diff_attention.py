"""diff_attention(): against the definition in 64 bits over sizes, head groups, layouts, key lengths and peaked rows; refusals.

Tolerance, per element. Probabilities are rounded to fp16 ahead of the second product: half a step, 2^-11 relative, and half of fp16's
smallest step, 2^-25, for those that small (relative to a maximum whose own probability is at least 1). Scores are fp32 sums of 64 exact
products, off by less than 64 * 2^-24 * sum |q k| * scale, which is what the exponent and so the probability is off by relatively
(times 1.45, with 2^-21 for the exponential and the fp32 sums): with these, map t's output is off by at most
  d_t = (2^-11 + e_t) A_t + 2^-25 S / l_t,   A_t = softmax-weighted |v|, S = sum |v|, l_t = sum of exp(score - maximum),  e_t the exponents'.
o is off by d = d_1 + |lam| d_2 (+ 2^-22 of |o_1| + |lam o_2| for the fp32 end). The norm y = o r w s, r = (mean o^2 + eps)^-1/2, is off by
|w s| r (d + |o| r rms(d)) to first order; a fifth more covers the second where r rms(d) < 0.1, which is checked. The result is rounded
to fp16: 2^-11 of it, or 2^-25."""
import pytest
import torch

from fastbb_b200 import _lib
from fastbb_b200.diff_attention import diff_attention


def reference(q, k, v, lam, weight=None, eps=1e-5, out_scale=1.0, scale=0.125, lengths=None):
    """(o, room) in 64 bits, room the tolerance."""
    B, Nq, H2, _ = q.shape
    H, Hk, Nk = H2 // 2, v.shape[2], k.shape[1]
    lam = lam.double().expand(B, Nq, H)
    o = torch.zeros(B, Nq, H, 128, dtype=torch.float64, device=q.device)
    d = torch.zeros_like(o)
    for b in range(B):
        n = Nk if lengths is None else min(max(int(lengths[b]), 0), Nk)
        for h in range(H if n else 0):
            vv = v[b, :n, h * Hk // H].double()
            for t in range(2):
                kk = k[b, :n, 2 * (h * Hk // H) + t].double()
                for lo in range(0, Nq, 1024):
                    qq = q[b, lo:lo + 1024, 2 * h + t].double()
                    s = qq @ kk.t() * scale
                    off = (qq.abs() @ kk.abs().t()).amax(-1, keepdim=True) * scale * 64 * 2.0 ** -24 * 1.45
                    p = torch.exp(s - s.amax(-1, keepdim=True))
                    l = p.sum(-1, keepdim=True)
                    x = p @ vv / l
                    dx = (2.0 ** -11 + 2 * off + 2.0 ** -21) * (p @ vv.abs() / l) + 2.0 ** -25 * vv.abs().sum(0) / l + 2.0 ** -22 * x.abs()
                    f = 1.0 if t == 0 else lam[b, lo:lo + 1024, h, None]
                    o[b, lo:lo + 1024, h] += x if t == 0 else -f * x
                    d[b, lo:lo + 1024, h] += dx if t == 0 else f.abs() * dx
    if weight is not None:
        r = (o.square().mean(-1, keepdim=True) + eps).rsqrt()
        rms = d.square().mean(-1, keepdim=True).sqrt() * r
        assert float(rms.max()) < 0.1
        d = 1.2 * weight.double().abs() * r * (d + o.abs() * rms)
        o = o * r * weight.double()
    o, d = o * out_scale, d * abs(out_scale)
    return o, d + o.abs() * 2.0 ** -11 + 2.0 ** -25


def check(got, *args, **kw):
    want, room = reference(*args, **kw)
    over = (got.double() - want).abs() - room
    assert bool((over <= 0).all()), f"{int((~(over <= 0)).sum())} of {over.numel()} off, worst by {float(over.max()):.3g}, room there {float(room.flatten()[over.argmax()]):.3g}"


def make(B, Nq, Nk, H, Hk, g, lam="head", std=1.0):
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    lam = torch.rand({"one": (), "head": (H,), "token": (B, Nq, H), "row": (Nq, 1)}[lam], generator=g, device="cuda") * 0.8
    return (rnd(B, Nq, 2 * H, 64) * std).half(), rnd(B, Nk, 2 * Hk, 64).half(), rnd(B, Nk, Hk, 128).half(), lam


@pytest.mark.gpu
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,lam,norm", [
    (1, 1, 1, 1, 1, "one", False), (1, 1, 127, 2, 1, "head", True), (2, 3, 128, 1, 1, "token", True), (1, 16, 129, 3, 1, "head", False),
    (2, 17, 64, 4, 2, "row", True), (1, 128, 128, 2, 2, "head", True), (1, 129, 257, 6, 6, "token", True), (2, 200, 300, 3, 3, "head", False),
    (1, 257, 257, 6, 2, "head", True), (1, 1, 5000, 3, 3, "head", True), (3, 5, 2049, 2, 1, "token", True), (1, 40, 16385, 1, 1, "one", True),
    (1, 500, 1500, 2, 2, "token", True), (9, 131, 384, 12, 4, "head", True), (1, 1041, 1041, 16, 16, "head", True), (2, 640, 7, 2, 2, "head", False)])
def test_matches_the_definition_in_64_bits(B, Nq, Nk, H, Hk, lam, norm):
    g = torch.Generator("cuda").manual_seed(Nq * 31 + Nk)
    q, k, v, lam = make(B, Nq, Nk, H, Hk, g, lam)
    weight = torch.randn(128, generator=g, device="cuda").mul_(0.2).add_(1)
    weight = None if not norm else weight.half() if Nq % 2 else weight
    out = diff_attention(q, k, v, lam, weight=weight, out_scale=0.8)
    check(out, q, k, v, lam, weight=weight, out_scale=0.8)
    assert torch.equal(out, diff_attention(q, k, v, lam, weight=weight, out_scale=0.8))  # the same bits again
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk,lengths", [(5, 400, [400, 0, 1, 128, 129, 399]), (300, 300, [300, 127, 0, 256, 255, 64]), (1, 4000, [3999, 4000, 0, 17, 2048, 2049]),
                                           (130, 129, [-3, 500, 129, 128, 65, 2])])
@pytest.mark.parametrize("bad", [0.0, float("nan"), float("inf")])
def test_keys_beyond_a_length_are_not_seen(Nq, Nk, lengths, bad):
    g = torch.Generator("cuda").manual_seed(Nk)
    q, k, v, lam = make(len(lengths), Nq, Nk, 2, 1, g, "token")
    weight = torch.randn(128, generator=g, device="cuda").half()
    for i, n in enumerate(lengths):
        if bad and n < Nk:
            k[i, max(n, 0):], v[i, max(n, 0):] = bad, -bad
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = diff_attention(q, k, v, lam, weight=weight, key_lengths=n)
    clean_k, clean_v = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
    check(out, q, clean_k, clean_v, lam, weight=weight, lengths=lengths)
    for i, m in enumerate(lengths):
        if m <= 0:
            assert bool((out[i] == 0).all())
    plain = diff_attention(q, k, v, lam, key_lengths=n, scale=0.3)
    check(plain, q, clean_k, clean_v, lam, lengths=lengths, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("B,Nq,Nk,H", [(7, 700, 700, 6), (40, 150, 200, 4), (33, 1, 300, 2)])
def test_many_tiles_of_uneven_lengths(B, Nq, Nk, H):
    """More tiles than SMs, some of no keys, their entries in no order; more entries than a warp has lanes."""
    g = torch.Generator("cuda").manual_seed(B)
    q, k, v, lam = make(B, Nq, Nk, H, H // 2, g)
    lengths = [(37 * i * i + 11) % (Nk + 1) if i % 3 else 0 for i in range(B)]
    weight = torch.randn(128, generator=g, device="cuda").half()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    check(diff_attention(q, k, v, lam, weight=weight, key_lengths=n), q, k, v, lam, weight=weight, lengths=lengths)
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [32, 40])
@pytest.mark.parametrize("keyed", ["first", "middle", "last", "both ends", "every seventh", "one in all"])
def test_long_runs_of_entries_without_keys(B, keyed):
    """Every CTA has many tiles in a row without keys, ahead of, between and behind those with some; in falling order of the lengths (32 entries) and in
    the entries' own (40). Rows beyond the queries' in every last tile."""
    g = torch.Generator("cuda").manual_seed(B)
    Nq, Nk, H = 1000, 130, 8
    q, k, v, lam = make(B, Nq, Nk, H, H // 2, g, "token")
    which = {"first": range(2), "middle": range(B // 2, B // 2 + 2), "last": range(B - 2, B), "both ends": (0, B - 1), "every seventh": range(0, B, 7),
             "one in all": (B // 3,)}[keyed]
    lengths = [(1, 64, 65, 130, 128, 17)[i % 6] if i in which else -(i % 2) for i in range(B)]
    weight = torch.randn(128, generator=g, device="cuda").half()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for _ in range(3):
        out = diff_attention(q, k, v, lam, weight=weight, key_lengths=n)
    rest = torch.tensor([m <= 0 for m in lengths], device="cuda")
    assert bool((out[rest] == 0).all())
    check(out[~rest], q[~rest], k[~rest], v[~rest], lam[~rest], weight=weight, lengths=[m for m in lengths if m > 0])
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.gpu
def test_thousands_of_tiles_without_keys():
    g = torch.Generator("cuda").manual_seed(1)
    q, k, v, lam = make(16, 2900, 0, 8, 8, g)
    out = torch.full((16, 2900, 8, 128), float("nan"), device="cuda", dtype=torch.float16)
    for _ in range(3):
        assert bool((diff_attention(q, k, v, lam, weight=torch.ones(128, device="cuda"), out=out) == 0).all())
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.gpu
def test_no_keys_at_all():
    g = torch.Generator("cuda").manual_seed(1)
    q, k, v, lam = make(2, 5, 0, 2, 2, g)
    out = torch.full((2, 5, 2, 128), float("nan"), device="cuda", dtype=torch.float16)
    assert bool((diff_attention(q, k, v, lam, out=out) == 0).all())
    assert diff_attention(q[:0], k[:0], v[:0], lam).shape == (0, 5, 2, 128) and diff_attention(q[:, :0], k, v, lam).shape == (2, 0, 2, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk", [(150, 700), (2, 3000)])
def test_maxima_that_rise_block_after_block(Nq, Nk):
    """Keys aligned with the queries and growing along the sequence: every block exceeds the running maximum by far more than 2^8."""
    g = torch.Generator("cuda").manual_seed(9)
    q, k, v, lam = make(1, Nq, Nk, 2, 2, g)
    q = (q * 0.2 + 1).half()
    k = (k * 0.1 + torch.linspace(0, 20, Nk, device="cuda")[None, :, None, None]).half()
    check(diff_attention(q, k, v, lam), q, k, v, lam)
    check(diff_attention(q, k.flip(1), v, lam), q, k.flip(1), v, lam)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["packed", "heads first", "wide"])
def test_strided_views_and_a_strided_output(layout):
    g = torch.Generator("cuda").manual_seed(4)
    B, N, H = 2, 205, 3
    if layout == "packed":
        buf = torch.randn(B, N, 6 * H * 64, generator=g, device="cuda").half()
        q, k, v = (t.view(B, N, -1, c) for t, c in zip(buf.split(2 * H * 64, -1), (64, 64, 128)))
    elif layout == "heads first":
        q, k = (torch.randn(B, 2 * H, N, 64, generator=g, device="cuda").half().transpose(1, 2) for _ in range(2))
        v = torch.randn(B, H, N, 128, generator=g, device="cuda").half().transpose(1, 2)
    else:
        q, k = (torch.randn(2 * B, N, 2 * H, 72, generator=g, device="cuda").half()[::2, ..., 8:] for _ in range(2))
        v = torch.randn(B, 2 * N, H, 128, generator=g, device="cuda").half()[:, 1::2]
    lam = torch.rand(H, N, B, generator=g, device="cuda").permute(2, 1, 0)
    frame = torch.full((B, N + 3, H + 1, 136), 7.0, device="cuda", dtype=torch.float16)
    out = diff_attention(q, k, v, lam, out=frame[:, 1:N + 1, :H, :128])
    check(out, q, k, v, lam)
    out.fill_(7.0)
    assert bool((frame == 7.0).all())  # nothing outside the rows was written


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    g = torch.Generator("cuda").manual_seed(5)
    far = 2 ** 31 + 4096
    store = torch.empty(far + 2 * 128 * 300, device="cuda", dtype=torch.float16)
    q, k, v, lam = make(2, 70, 150, 1, 1, g)
    kb = store.as_strided((2, 150, 2, 64), (far, 128, 64, 1))
    vb = store.as_strided((2, 150, 1, 128), (far, 128, 128, 1), 128 * 150)
    ob = torch.empty(far + 128 * 70, device="cuda", dtype=torch.float16).as_strided((2, 70, 1, 128), (far, 128, 128, 1))
    kb.copy_(k)
    vb.copy_(v)
    check(diff_attention(q, kb, vb, lam, out=ob), q, k, v, lam)


@pytest.mark.gpu
def test_other_stream_and_graphs_that_live_side_by_side():
    g = torch.Generator("cuda").manual_seed(6)
    sets = [make(1, n, m, 4, 4, g) for n, m in ((3, 3000), (260, 260), (1, 6000))]
    want = [diff_attention(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [diff_attention(*s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, diff_attention(*s)))
    for _ in range(2):
        for (graph, out), w in zip(graphs, want):
            out.zero_()
            graph.replay()
    for o, (_, c), w in zip(other, graphs, want):
        assert torch.equal(o, w) and torch.equal(c, w)


@pytest.mark.gpu
def test_with_one_map_off_it_is_attention():
    """lam = 0 leaves the first map: what attention() gives for each half of the values. Both round the same probabilities to fp16."""
    from fastbb_b200.attention import attention
    g = torch.Generator("cuda").manual_seed(8)
    q, k, v, _ = make(1, 390, 390, 2, 2, g)
    out = diff_attention(q, k, v, torch.zeros((), device="cuda"))
    for half in (0, 64):
        one = attention(q[:, :, ::2], k[:, :, ::2], v[..., half:half + 64])
        assert float((out[..., half:half + 64].float() - one.float()).abs().max()) <= 2.0 ** -9


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk", [(3, 4000), (200, 300)])
def test_rows_without_keys_are_zero_with_a_norm_of_no_epsilon(Nq, Nk):
    """Few queries over many keys (two launches) and tiles of one launch alike."""
    g = torch.Generator("cuda").manual_seed(Nq)
    q, k, v, lam = make(3, Nq, Nk, 2, 2, g)
    weight = torch.randn(128, generator=g, device="cuda").half()
    lengths = [Nk, 0, 70]
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = diff_attention(q, k, v, lam, weight=weight, eps=0.0, key_lengths=n)
    assert bool((out[1] == 0).all())
    check(out[::2], q[::2], k[::2], v[::2], lam, weight=weight, eps=0.0, lengths=lengths[::2])


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk,dead", [(200, 300, 64), (200, 300, 299), (1, 4000, 700), (5, 129, 128), (3, 4000, 3999)])
def test_scores_of_minus_infinity_ahead_of_the_others(Nq, Nk, dead):
    """Keys that an infinity in them takes out of every row's maps have no weight, whole blocks and shares of them too; a row of nothing else is NaN."""
    g = torch.Generator("cuda").manual_seed(dead)
    q, k, v, lam = make(2, Nq, Nk, 2, 2, g)
    q[..., 5] = 0.5 + q[..., 5].abs()
    kept = slice(dead, Nk)
    k[:, :dead, :, 5] = -float("inf")
    out = diff_attention(q, k, v, lam)
    check(out, q, k[:, kept], v[:, kept], lam)
    k[1, :, :, 5] = -float("inf")
    out = diff_attention(q, k, v, lam)
    assert bool(out[1].isnan().all())
    check(out[:1], q[:1], k[:1, kept], v[:1, kept], lam)
    assert _lib.device_status() == (0, 0, 0, 0)


FAR = {  # (first column of a key, second column): with queries of 2^15 and 2^7 there, scores of 2^15 times the first and 2^7 times the second
    "rising": lambda j, n: (torch.floor(16.0 * j / n) * 4000 - 2000, j % 5),
    "falling": lambda j, n: (60000 - torch.floor(16.0 * j / n) * 4000, j % 7),
    "ties": lambda j, n: (60000 + 0 * j, 0 * j),
    "near ties": lambda j, n: (48000 + 0 * j, j % 3),
    "far below nought": lambda j, n: (-60000 + 32 * (j % 11), 0 * j),
    "from far below to near": lambda j, n: (torch.where(j < 0.7 * n, -50000.0, 0.0), j % 4),
    "near, then far, then further": lambda j, n: (torch.where(j < 0.3 * n, 0.0, torch.where(j < 0.6 * n, 3000.0, 40000.0)), j % 2),
    "around 2^22": lambda j, n: (700 + torch.floor(8.0 * j / n), j % 6),
}


@pytest.mark.gpu
@pytest.mark.parametrize("Nq,Nk,scale", [(150, 300, None), (1, 3000, None), (20, 129, 1.0), (5, 2500, 3e-5), (3, 500, 1e27)])
@pytest.mark.parametrize("kind", FAR)
def test_scores_of_any_magnitude(Nq, Nk, scale, kind):
    """Scores that fp32 holds exactly, so that they have no tolerance, up to 3e8 times scale and far apart. Tolerance: exponents are differences of
    exact scores times scale, off by 2^-22 of themselves; those of weights that count are below 32: 2^-17. The rest as above."""
    g = torch.Generator("cuda").manual_seed(Nk)
    j = torch.arange(Nk, device="cuda", dtype=torch.float64)
    first, second = FAR[kind](j, Nk)
    q, k = torch.zeros(1, Nq, 4, 64, device="cuda").half(), torch.zeros(1, Nk, 4, 64, device="cuda").half()
    q[..., 3], q[..., 40] = 2.0 ** 15, 2.0 ** 7
    q[:, ::2, 1] = 0  # some rows of all scores alike, beside the far ones
    for head in range(4):
        turn = head * (Nk // 5)  # each map meets its maxima elsewhere
        k[0, :, head, 3], k[0, :, head, 40] = first.roll(turn).half(), second.roll(turn).half()
    v, lam = torch.randn(1, Nk, 2, 128, generator=g, device="cuda").half(), torch.tensor([0.3, 0.6], device="cuda")
    s_ = 0.125 if scale is None else float(torch.tensor(scale))
    want, room = torch.zeros(1, Nq, 2, 128, dtype=torch.float64, device="cuda"), 0
    for t in range(2):
        s = torch.einsum("qhc,khc->hqk", q[0, :, t::2].double(), k[0, :, t::2].double())
        assert torch.equal(s.float().double(), s)
        p = torch.exp((s - s.amax(-1, keepdim=True)) * s_)
        l = p.sum(-1, keepdim=True)
        vv = v[0].double().transpose(0, 1)
        x, f = (p @ vv / l).transpose(0, 1), 1.0 if t == 0 else lam.double()[:, None]
        d = ((2.0 ** -11 + 2.0 ** -16 + 2.0 ** -21) * (p @ vv.abs() / l) + 2.0 ** -25 * vv.abs().sum(1, keepdim=True) / l).transpose(0, 1) + 2.0 ** -22 * x.abs()
        want[0] += x if t == 0 else -f * x
        room = room + f * d
    out = diff_attention(q, k, v, lam, scale=scale)
    over = (out[0].double() - want[0]).abs() - room - want[0].abs() * 2.0 ** -11 - 2.0 ** -25
    assert bool((over <= 0).all()), f"{int((~(over <= 0)).sum())} of {over.numel()} off, worst by {float(over.max()):.3g}"
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    g = torch.Generator("cuda").manual_seed(7)
    q, k, v, lam = make(2, 20, 30, 4, 2, g)
    n = torch.tensor([30, 30], dtype=torch.int32, device="cuda")
    for call in (
            lambda: diff_attention(q.float(), k, v, lam), lambda: diff_attention(q, k[..., :32], v, lam), lambda: diff_attention(q, k, v[..., :64], lam),
            lambda: diff_attention(q[:, :, :7], k, v, lam), lambda: diff_attention(q[:, :, :6], k, v, lam), lambda: diff_attention(q, k, v[:, :29], lam),
            lambda: diff_attention(q, k[:1], v[:1], lam), lambda: diff_attention(q, k[:1].expand(2, 30, 4, 64), v, lam),
            lambda: diff_attention(q, k, v, lam.half()), lambda: diff_attention(q, k, v, 0.5), lambda: diff_attention(q, k, v, lam[:3]),
            lambda: diff_attention(q, k, v, lam.cpu()), lambda: diff_attention(q, k, v, lam, scale=0.0), lambda: diff_attention(q, k, v, lam, scale=float("nan")),
            lambda: diff_attention(q, k, v, lam, eps=-1.0), lambda: diff_attention(q, k, v, lam, weight=torch.ones(64, device="cuda")),
            lambda: diff_attention(q, k, v, lam, weight=torch.ones(128, device="cuda").bfloat16()), lambda: diff_attention(q, k, v, lam, key_lengths=n.long()),
            lambda: diff_attention(q, k, v, lam, key_lengths=n[:1]), lambda: diff_attention(q, k, v, lam, out=torch.empty(2, 20, 4, 64, device="cuda").half()),
            lambda: diff_attention(q, k, v, lam, out=q.view(2, 20, 4, 128)),
            lambda: diff_attention(q, k, v, lam, out=torch.empty(1, 20, 4, 128, device="cuda").half().expand(2, 20, 4, 128)),
            lambda: diff_attention(torch.empty(2, 20, 8, 65, device="cuda").half()[..., 1:], k, v, lam)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_outputs_over_any_input_are_refused():
    """out shares 16 bytes with one input at a time; right behind it the call is taken."""
    g = torch.Generator("cuda").manual_seed(8)
    q, k, v, lam = make(2, 20, 30, 2, 1, g, "token")
    parts = dict(q=q, k=k, v=v, lam=lam, weight=torch.ones(128, device="cuda"), lengths=torch.tensor([30, 7], dtype=torch.int32, device="cuda"))
    size = 2 * q.numel() // 64 * 64
    store = torch.zeros(1 << 18, dtype=torch.uint8, device="cuda")
    for name, t in parts.items():
        n = t.numel() * t.element_size()
        view = store[:n].view(t.dtype).view(t.shape)
        view.copy_(t)
        use = {**parts, name: view}
        call = lambda lo: diff_attention(use["q"], use["k"], use["v"], use["lam"], weight=use["weight"], key_lengths=use["lengths"],  # noqa: E731, B023
                                         out=store[lo:lo + size].view(torch.float16).view(2, 20, 2, 128))
        clear, held = (n + 15) // 16 * 16, store.clone()
        with pytest.raises(ValueError, match="shares memory"):
            call(clear - 16)
        assert torch.equal(store, held)
        call(clear)


@pytest.mark.gpu
def test_factors_that_fp32_does_not_hold_are_refused():
    g = torch.Generator("cuda").manual_seed(7)
    q, k, v, lam = make(1, 4, 6, 2, 2, g)
    for bad in ({"scale": 1e39}, {"scale": float("inf")}, {"eps": 1e39}, {"eps": float("nan")}, {"out_scale": -1e39}, {"out_scale": float("inf")}):
        with pytest.raises(ValueError, match="finite"):
            diff_attention(q, k, v, lam, **bad)
    for good in ({"scale": 3e38}, {"eps": 3e38}, {"out_scale": -3e38}, {"out_scale": 0.0}):
        diff_attention(q, k, v, lam, **good)


# ------------------------------------------------------------------------------------------------------------------ CPU
def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 4, 2, 64).half()
    with pytest.raises(ValueError, match="no fallback"):
        diff_attention(q, q, torch.zeros(1, 4, 1, 128).half(), torch.zeros(()))


def test_entry_point_refusals():
    lib, A = _lib.load(), 0x7F0000000000

    def call(q=A, k=A, v=A, o=A, B=2, Nq=4, Nk=6, H=4, Hk=2, st=None, lam=A, weight=A, wd=0, eps=1e-5, scale=0.125, ws=None):
        st = st or [2048, 512, 64, 2048, 256, 64, 2048, 256, 128, 2048, 512, 128]
        return lib.fbb_diff64_f16(q, k, v, o, B, Nq, Nk, H, Hk, *st, lam, 0, 0, 1, weight, wd, eps, 1.0, scale, None, ws, 0, None)

    assert call(q=None) == call(o=None) == call(lam=None) == call(k=None) == call(v=None) == -1
    assert call(B=-1) == call(H=0) == call(Hk=3) == call(Hk=0) == call(scale=0.0) == call(scale=float("nan")) == call(eps=-1.0) == -2
    assert call(q=A + 8) == call(o=A + 2) == call(ws=A + 4) == -3
    for i in range(12):
        for value in (0, 12, -64):
            st = [2048, 512, 64, 2048, 256, 64, 2048, 256, 128, 2048, 512, 128]
            st[i] = value
            assert call(st=st) == -3, (i, value)
    assert call(wd=1) == call(wd=7) == -4
    assert call(B=0, q=None) == call(Nq=0, o=None) == 0
    assert lib.fbb_diff64_workspace_bytes(0, 1, 1000, 8) == 0 and lib.fbb_diff64_launches(1, 0, 10, 2) == 0


def test_the_record_form_refuses_what_the_other_does():
    """Every field is where the entry point looks for it: broken alone, it is the one that is named."""
    lib, A = _lib.load(), 0x7F0000000000
    good = dict(q=A, k=A, v=A, o=A, lam=A, weight=A, lengths=A, ws=0, stream=0, **{f"s{i}": n for i, n in enumerate((2048, 512, 64, 2048, 256, 64, 2048, 256, 128, 2048, 512, 128))},
                l0=0, l1=0, l2=1, need=0, B=2, Nq=4, Nk=6, H=4, Hk=2, wd=0, eps=1e-5, out_scale=1.0, scale=0.125)

    def call(**kw):
        return lib.fbb_diff64_f16_from(_lib.Diff64Args.pack(*{**good, **kw}.values()))

    assert lib.fbb_diff64_f16_from(None) == call(q=0) == call(k=0) == call(v=0) == call(o=0) == call(lam=0) == -1
    assert call(B=-1) == call(Nq=-1) == call(Nk=-1) == call(H=0) == call(Hk=3) == call(scale=0.0) == call(eps=-1.0) == -2 and call(wd=7) == -4
    assert [call(**{f"s{i}": 12}) for i in range(12)] == [-3] * 12 and call(ws=A + 4) == -3 and call(weight=0, wd=7, Nq=0) == call(B=0, q=0) == 0
    many = dict(B=1, Nq=1, Nk=4096, H=1, Hk=1)  # (split over the keys: the workspace is asked for)
    assert call(**many, ws=A, need=lib.fbb_diff64_workspace_bytes(1, 1, 4096, 1) - 1) == -2 and b"workspace" in lib.fbb_last_error()
