"""GPU: sampling against its definition in 64 bits (ids equal, log-probabilities within rounding)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def draw64(x, u, t, k, p, m):
    """One row: (id, logprob) from the definition; ``x`` doubles."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return 0, math.nan
    if not t > 0:
        return int(np.argmax(x)), 0.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / t))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if 0 < k < len(order):
        order = order[: int(k)]
    if p < 1:
        c = np.concatenate([[0.0], np.cumsum(w[order])])
        order = order[: max(1, int((c[:-1] < max(p, 0.0) * c[-1]).sum()))]
    if m > 0:
        order = order[: max(1, int((w[order] >= m).sum()))]
    kept = np.sort(order)
    c = np.cumsum(w[kept])
    at = min(int(np.searchsorted(c, u * c[-1], side="right")), len(kept) - 1)
    return int(kept[at]), math.log(w[kept[at]] / c[-1]) if w[kept[at]] > 0 else -math.inf


def check(logits, uniform, knobs, dev, **kw):
    from prime_kernels_b200 import sampling as S

    rows = logits.shape[0]
    ids, lp = S.sample(logits, uniform.to(dev), return_logprobs=True,
                       **{n: (v.to(dev) if torch.is_tensor(v) else v) for n, v in knobs.items()}, **kw)
    full = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **knobs}
    at = lambda v, r: float(v[r]) if torch.is_tensor(v) else float(np.float32(v))      # noqa: E731
    x = logits.double().cpu().numpy()
    for r in range(rows):
        want, wlp = draw64(x[r], float(uniform[r]), *(at(full[n], r) for n in ("temperature", "top_k", "top_p", "min_p")))
        assert int(ids[r]) == want, (r, int(ids[r]), want)
        # a double rounded to fp32 (2^-24 of it); weights to 2^-44 of the largest: nothing beside that
        assert abs(float(lp[r]) - wlp) <= 2 ** -23 * abs(wlp) + 1e-9 or (math.isnan(wlp) and math.isnan(float(lp[r])))
    return ids


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 49152), (5, 1000), (3, 33), (2, 2), (4, 1), (40, 4099), (90, 517), (200, 257)])
@pytest.mark.parametrize("knobs", [
    {}, {"top_k": 7}, {"top_p": 0.8}, {"min_p": 0.1}, {"temperature": 0.0},
    {"temperature": 0.7, "top_k": 50, "top_p": 0.9, "min_p": 0.01}, {"temperature": 1.7, "top_k": 300, "top_p": 0.5}])
def test_types_sizes_filters(cuda_device, dtype, rows, vocab, knobs):
    g = torch.Generator().manual_seed(rows * 1000 + vocab)
    x = (torch.randn(rows, vocab, generator=g) * 2).to(TYPES[dtype]).to(cuda_device)
    check(x, torch.rand(rows, generator=g), knobs, cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("levels", [1, 2, 5])
@pytest.mark.parametrize("knobs", [{"top_k": 100}, {"top_p": 0.37}, {"top_k": 2000, "top_p": 0.9}, {"top_k": 1}])
def test_ties_go_to_the_lowest_index(cuda_device, dtype, levels, knobs):
    """Few distinct logits: the border of every filter falls among equal tokens."""
    g = torch.Generator().manual_seed(levels)
    x = torch.randint(0, levels, (6, 5003), generator=g).to(TYPES[dtype]).to(cuda_device)
    check(x, torch.rand(6, generator=g), knobs, cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
def test_settings_of_each_row(cuda_device, dtype):
    g = torch.Generator().manual_seed(5)
    rows, vocab = 64, 3001
    x = (torch.randn(rows, vocab, generator=g) * 3).to(TYPES[dtype]).to(cuda_device)
    i = torch.arange(rows)
    knobs = {"temperature": torch.where(i % 5 == 0, torch.zeros(rows), 0.3 + i / 40).float(),
             "top_k": torch.where(i % 3 == 0, torch.full((rows,), -1), i * 7 + 1).int(),
             "top_p": torch.where(i % 4 == 0, torch.full((rows,), 1.5), (i + 1) / 66).float(),
             "min_p": torch.where(i % 2 == 0, torch.full((rows,), -1.0), i / 500).float()}
    knobs["temperature"][10], knobs["temperature"][11] = -1.0, math.nan
    knobs["top_p"][21], knobs["top_p"][22] = -0.5, 0.0
    knobs["min_p"][31] = 1.0
    check(x, torch.rand(rows, generator=g), knobs, cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("knobs", [{}, {"top_k": 3}, {"top_k": 1}, {"top_k": 600}, {"top_p": 0.6}, {"min_p": 0.2}, {"min_p": 1.0}, {"temperature": 0.0}])
def test_masked_and_special_logits(cuda_device, dtype, knobs):
    g = torch.Generator().manual_seed(8)
    t, vocab = TYPES[dtype], 700
    low = torch.finfo(t).min
    rows = []

    def row(fill, **at):
        x = torch.full((vocab,), fill) if fill is not None else torch.randn(vocab, generator=g)
        for i, v in at.items():
            x[int(i[1:])] = v
        rows.append(x)

    row(-math.inf)                                     # nothing left: id 0, NaN
    row(math.nan)
    row(-math.inf, i699=1.0)                           # one token left
    row(math.nan, i350=-5.0, i12=-math.inf)
    row(-math.inf, i5=2.0, i300=2.0, i301=1.0)
    row(low)                                           # the type's lowest value everywhere: all equal
    row(low, i77=0.0, i78=0.5)                         # a mask of lowest values
    row(None, i3=math.inf)                             # one infinity takes everything
    row(None, i3=math.inf, i600=math.inf)
    row(math.inf)
    row(-math.inf, i8=math.inf, i7=math.inf, i9=math.nan)
    row(0.0, i9=-0.0, i10=-0.0)                        # signed zeros are equal
    row(-0.0, i400=0.0)
    row(None, i0=math.nan, i699=-math.inf)
    x = torch.stack(rows).to(t).to(cuda_device)
    for u in (0.0, 0.3, 0.7, 1 - 2 ** -24):
        check(x, torch.full((len(rows),), u), knobs, cuda_device)


@pytest.mark.parametrize("temperature", [1e-40, 1e-30, 1e-3, 0.02, 0.1, 0.4])
@pytest.mark.parametrize("knobs", [{"top_p": 0.9}, {"top_k": 50}, {"top_k": 1000}, {"top_k": 50, "top_p": 0.7}, {"top_k": 1000, "top_p": 0.95},
                                   {"top_k": 20000, "top_p": 0.999, "min_p": 1e-6}])
def test_low_temperatures(cuda_device, temperature, knobs):
    """Most of a row far below the weights that count, and border bins many times a binade wide."""
    g = torch.Generator().manual_seed(int(1 / temperature) % 1000)
    x = torch.randn(6, 30011, generator=g) * torch.tensor([0.2, 1.0, 3.0, 3.0, 6.0, 60.0])[:, None]
    check(x.bfloat16().to(cuda_device), torch.rand(6, generator=g), {"temperature": temperature, **knobs}, cuda_device)
    check(x.to(cuda_device), torch.rand(6, generator=g), {"temperature": temperature, **knobs}, cuda_device)


def test_uniform_borders(cuda_device):
    """u = 0 draws the first kept token however small its weight, u next to 1 the last one that moves the sum."""
    from prime_kernels_b200 import sampling as S

    x = torch.tensor([[-30.0, 0.0, -30.0], [-25.0, -25.0, 0.0], [0.0, 0.0, 0.0]], device=cuda_device)
    assert S.sample(x, torch.zeros(3, device=cuda_device)).tolist() == [0, 0, 0]
    assert S.sample(x, torch.full((3,), 1 - 2 ** -24, device=cuda_device)).tolist() == [1, 2, 2]
    # out-of-range numbers are taken as the nearest one inside
    assert S.sample(x, torch.tensor([-1.0, math.nan, 2.0], device=cuda_device)).tolist() == [0, 0, 2]


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_largest_vocabulary(cuda_device, dtype):
    from prime_kernels_b200 import sampling as S

    g = torch.Generator().manual_seed(3)
    wide = torch.randn(9, 1201, generator=g).to(TYPES[dtype]).to(cuda_device)
    check(wide[::2, 1:1200], torch.rand(5, generator=g), {"top_k": 40, "top_p": 0.9}, cuda_device)   # rows at odd addresses
    big = torch.randn(2, S.MAX_VOCAB, generator=g).to(TYPES[dtype]).to(cuda_device)
    check(big, torch.rand(2, generator=g), {"top_k": 60000, "top_p": 0.95}, cuda_device)
    one = torch.randn(1, 3000, generator=g).to(TYPES[dtype]).to(cuda_device).expand(4, 3000)         # rows that share storage
    check(one, torch.rand(4, generator=g), {"top_p": 0.9}, cuda_device)


def test_the_same_whatever_the_batch(cuda_device):
    """A row's draw does not depend on how many rows share the call (the rows are spread differently)."""
    from prime_kernels_b200 import sampling as S

    g = torch.Generator(device=cuda_device).manual_seed(4)
    x = torch.randn(300, 49152, generator=g, device=cuda_device).to(torch.bfloat16)
    u = torch.rand(300, generator=g, device=cuda_device)
    kw = dict(temperature=0.9, top_k=1000, top_p=0.97, return_logprobs=True)
    ids, lp = S.sample(x, u, **kw)
    for a, b in ((0, 1), (5, 30), (17, 60), (100, 174)):
        i, l = S.sample(x[a:b], u[a:b], **kw)
        assert torch.equal(i, ids[a:b]) and torch.equal(l, lp[a:b])


def test_frequencies(cuda_device):
    """2^20 draws from eight tokens: counts within six standard deviations of the softmax."""
    from prime_kernels_b200 import sampling as S

    n = 1 << 20
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5, -3.0, 1.5, -0.5])
    g = torch.Generator(device=cuda_device).manual_seed(6)
    u = torch.rand(n, generator=g, device=cuda_device)
    got = torch.bincount(S.sample(x.to(cuda_device).expand(n, 8), u, temperature=1.0), minlength=8).double().cpu()
    p = torch.softmax(x.double(), 0)
    assert ((got - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt()).all()


def test_out_streams_and_graphs(cuda_device):
    from prime_kernels_b200 import sampling as S

    g = torch.Generator(device=cuda_device).manual_seed(2)
    x = torch.randn(8, 4099, generator=g, device=cuda_device)
    u = torch.rand(8, generator=g, device=cuda_device)
    kw = dict(temperature=0.8, top_k=50, top_p=0.9)
    want = S.sample(x, u, **kw)
    out = torch.full((8,), -7, dtype=torch.int64, device=cuda_device)
    assert S.sample(x, u, out=out, **kw) is out and torch.equal(out, want)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        S.sample(x, u, out=out, **kw)
        with torch.cuda.graph(graph, stream=side):
            S.sample(x, u, out=out, **kw)
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    x2 = torch.randn(8, 4099, generator=g, device=cuda_device)
    want2 = S.sample(x2, u, **kw)
    x.copy_(x2)
    graph.replay()
    assert torch.equal(out, want2)
    assert S.sample(x[:0], u[:0]).shape == (0,)


def test_refusals(cuda_device):
    from prime_kernels_b200 import sampling as S

    x, u = torch.zeros(2, 16, device=cuda_device), torch.zeros(2, device=cuda_device)
    for kw in ({"temperature": -1.0}, {"temperature": math.inf}, {"temperature": math.nan}, {"top_k": -1}, {"top_p": 0.0},
               {"top_p": 1.1}, {"min_p": -0.1}, {"min_p": 1.5}):
        with pytest.raises(ValueError):
            S.sample(x, u, **kw)
    bad = [(x.double(), u, {}), (x[0], u, {}), (x.t(), u, {}), (x, u.double(), {}), (x, u[:1], {}), (x, u.cpu(), {}),
           (x, u, {"top_k": torch.zeros(2, dtype=torch.int64, device=cuda_device)}),
           (x, u, {"temperature": torch.zeros(3, device=cuda_device)}), (x, u, {"top_p": torch.zeros(2)}),
           (x, u, {"out": torch.zeros(2, dtype=torch.int32, device=cuda_device)}),
           (torch.zeros(1, S.MAX_VOCAB + 1, device=cuda_device), u[:1], {}), (x[:, :0], u, {})]
    for logits, uniform, kw in bad:
        with pytest.raises(RuntimeError):
            S.sample(logits, uniform, **kw)
    with pytest.raises(NotImplementedError):
        S.sample(x.cpu(), u.cpu())


def test_session_draws_from_its_logits(cuda_device):
    """DecodeSession with a sampler: temperature 0 repeats the greedy run; otherwise each id is the draw from that
    step's logits and is what the next step is fed."""
    from prime_kernels_b200 import decode as D
    from prime_kernels_b200 import harness
    from prime_kernels_b200 import sampling as S

    geom = D.Geometry("sampled", 192, 512, 2, 3, 1, vocab=1024)
    wd = harness.weights_to(harness.make_weights(geom, 0, norm_weights="random", std=0.2), cuda_device)
    cs = harness.make_cos_sin_cache(geom, 64, cuda_device)

    def run(sampler):
        kv = harness.PagedKV(geom, 2, 64, cuda_device)
        ses = D.DecodeSession(geom, embed=wd["embed"], layers=wd["layers"], final_norm=wd["final_norm"],
                              kv_caches=kv.kv_caches, cos_sin_cache=cs, block_table=kv.block_table)
        ses.start(torch.tensor([5, 700]), torch.tensor([0, 0]))
        return ses.generate(12, collect_logits=True, sampler=sampler)

    greedy, logits = run(None)
    same, _ = run(S.Sampler(temperature=0.0))
    assert torch.equal(greedy, same)
    gen = torch.Generator(device=cuda_device).manual_seed(9)
    ids, logits = run(S.Sampler(temperature=1.5, top_p=0.9, generator=gen))
    gen.manual_seed(9)
    for t in range(12):
        u = torch.rand(2, generator=gen, device=cuda_device)
        assert torch.equal(S.sample(logits[t], u, temperature=1.5, top_p=0.9), ids[t])
    assert not torch.equal(ids, greedy)
    # fed back: a second run that forces those ids reproduces the logits of the sampled run
    kv = harness.PagedKV(geom, 2, 64, cuda_device)
    ses = D.DecodeSession(geom, embed=wd["embed"], layers=wd["layers"], final_norm=wd["final_norm"], kv_caches=kv.kv_caches,
                          cos_sin_cache=cs, block_table=kv.block_table)
    ses.start(torch.tensor([5, 700]), torch.tensor([0, 0]))
    for t in range(12):
        _, l, _ = ses.step()
        assert torch.equal(l, logits[t])
        ses.input_ids.copy_(ids[t])
