"""Tokens drawn from logits (plamo_kernel_sample) against a 64-bit implementation.

Tokens have to be equal.  The kernel's sums are off the 64-bit ones by about 2^-46 of the largest weight
for each token, so a number would have to fall within some 1e-9 of a border to be told otherwise: none of
the seeds here does."""
import numpy as np
import pytest
import torch

from paged_common import TYPES, lib, sample, sample64

pytestmark = pytest.mark.gpu


def controls(rng, rows, **fixed):
    c = {"temperature": rng.uniform(0.3, 1.7, rows), "top_k": rng.integers(1, 60, rows), "top_p": rng.uniform(0.2, 0.999, rows),
         "min_p": rng.uniform(0.0005, 0.2, rows)}
    c.update({k: np.full(rows, v) for k, v in fixed.items()})
    return {k: v.astype(np.int32 if k == "top_k" else np.float32) for k, v in c.items()}


def check(logits, uniform, **c):
    """`logits` a (strided) tensor on the GPU; controls as arrays, absent ones off."""
    rows, n = logits.shape
    uniform = np.asarray(uniform, np.float32)
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    token, prob = sample(logits, n, put(uniform), **{k: put(v) for k, v in c.items()})
    torch.cuda.synchronize()
    assert token[rows] == -7 and prob[rows] == -7
    x = logits.double().cpu().numpy()
    for r in range(rows):
        own = {k: float(v[r]) if k != "top_k" else int(v[r]) for k, v in c.items()}
        want, share = sample64(x[r], min(max(float(uniform[r]), 0.0), 1.0), **own)
        assert int(token[r]) == want, (r, own, float(uniform[r]), int(token[r]), want)
        assert abs(float(prob[r]) - share) <= 2.0 ** -23 * share + 1e-12, (r, own)
    return token[:rows].clone(), prob[:rows].clone()


def bell(rng, rows, n, kind, std=2.5, peaks=8):
    x = rng.standard_normal((rows, n)) * std
    for r in range(rows):
        x[r, rng.integers(0, n, peaks)] += rng.uniform(0, 11, peaks)
    return torch.from_numpy(x).to(TYPES[kind]).cuda()


MIXES = {"all": {}, "top_k": {"top_p": 1.0, "min_p": 0.0}, "top_p": {"top_k": 0, "min_p": 0.0},
         "min_p": {"top_k": 0, "top_p": 1.0}, "none": {"top_k": 0, "top_p": 1.0, "min_p": 0.0},
         "many_k": {"top_k": 5000, "min_p": 0.0}, "greedy": {"temperature": 0.0}, "hot": {"temperature": 30.0, "top_k": 0}}


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("mix", sorted(MIXES))
def test_controls(kind, mix):
    rng = np.random.default_rng([len(mix), len(kind)])
    for rows, n in ((9, 107520), (5, 20001)):
        check(bell(rng, rows, n, kind), rng.random(rows), **controls(rng, rows, **MIXES[mix]))


@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 9, 63, 64, 65, 1000, 1023, 4097])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_small_vocabularies_in_rows_of_any_alignment(n, kind):
    rng = np.random.default_rng(n)
    for pad in (0, 1, 5):
        wide = torch.full((6, n + pad), 1e30 if kind == "fp32" else 1e30, dtype=TYPES[kind], device="cuda")
        wide[:, :n] = bell(rng, 6, n, kind)
        check(wide[:, :n], rng.random(6), **controls(rng, 6))
        check(wide[:, :n], rng.random(6))


def test_largest_vocabulary_and_many_rows():
    rng = np.random.default_rng(5)
    check(bell(rng, 2, 1 << 20, "bf16"), rng.random(2), **controls(rng, 2, top_k=0))
    check(bell(rng, 2, (1 << 20) - 3, "fp32"), rng.random(2))
    check(bell(rng, 700, 513, "fp16"), rng.random(700), **controls(rng, 700))


def test_absent_controls():
    rng = np.random.default_rng(6)
    x, c = bell(rng, 4, 5000, "bf16"), controls(rng, 4)
    for names in ((), ("temperature",), ("top_k",), ("top_p",), ("min_p",), ("top_k", "top_p")):
        check(x, rng.random(4), **{k: c[k] for k in names})
    u = torch.full((4,), 0.5, device="cuda")
    a, _ = sample(x, 5000, u)
    b, none = sample(x, 5000, u, prob=False)
    assert none is None and torch.equal(a, b)


def test_controls_at_their_ends():
    rng = np.random.default_rng(7)
    x = bell(rng, 3, 3000, "fp32")
    u = [0.0, 0.5, 1 - 2.0 ** -24]
    for c in ({"top_k": 1}, {"top_k": 3000}, {"top_k": 2 ** 31 - 1}, {"top_k": -5}, {"top_p": 0.0}, {"top_p": -1.0},
              {"top_p": 2.0}, {"top_p": 1e-30}, {"top_p": 1 - 2.0 ** -24}, {"min_p": 1.0}, {"min_p": 7.0}, {"min_p": -1.0},
              {"min_p": 1e-12}, {"temperature": -1.0}, {"temperature": 1e-30}, {"temperature": 1e30}, {"temperature": 1e-3}):
        full = controls(rng, 3, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, **{})
        full.update({k: np.full(3, v, np.int32 if k == "top_k" else np.float32) for k, v in c.items()})
        check(x, u, **full)
    # numbers outside [0, 1) draw as its ends do; NaN controls and numbers as if off, and as 0
    one = lambda v: torch.full((3,), v, device="cuda")  # noqa: E731
    low, high = sample(x, 3000, one(0.0))[0], sample(x, 3000, one(1.0))[0]
    assert torch.equal(sample(x, 3000, one(-3.0))[0], low) and torch.equal(sample(x, 3000, one(9.0))[0], high)
    nan = float("nan")
    assert torch.equal(sample(x, 3000, one(nan), top_p=one(nan), min_p=one(nan))[0], low)
    assert torch.equal(sample(x, 3000, one(0.5), temperature=one(nan))[0][:3].cpu(), x.argmax(1).int().cpu())


def test_equal_logits():
    """Ties go to the lowest id, in the top-k as in the order of the draw."""
    for n in (10, 2048, 2049, 50000):
        x = torch.zeros(8, n, device="cuda")
        u = np.arange(8) / 8 + 0.03
        check(x, u)
        check(x, u, top_k=np.full(8, n // 2, np.int32))
        check(x, u, top_p=np.full(8, 0.5, np.float32))
    x = torch.full((8, 30000), -3.0, device="cuda")
    x[:, ::3] = 1.0                      # 10,000 equal ones above 20,000
    x[:, 7] = 1.5
    for k in (1, 2, 700, 9999, 10001, 10002, 25000):
        check(x.to(torch.bfloat16), np.arange(8) / 8 + 0.01, top_k=np.full(8, k, np.int32))
    check(x, np.arange(8) / 8 + 0.01, top_p=np.linspace(0.1, 0.99, 8).astype(np.float32))
    zero = torch.zeros(2, 100, device="cuda")
    zero[:, ::2] = -0.0
    assert sample(zero, 100, torch.zeros(2, device="cuda"))[0][:2].tolist() == [0, 0]


def test_logits_closer_than_a_bin():
    """Tens of thousands of values within a thousandth: borders are found by dividing a bin again."""
    rng = np.random.default_rng(8)
    x = torch.from_numpy(rng.standard_normal((6, 60000)) * 1e-4 + 5).float().cuda()
    u = rng.random(6)
    check(x, u)
    check(x, u, top_k=rng.integers(1, 60000, 6).astype(np.int32))
    check(x, u, top_p=rng.uniform(0.1, 0.95, 6).astype(np.float32))
    check(x, u, top_k=rng.integers(20000, 60000, 6).astype(np.int32), top_p=rng.uniform(0.3, 0.9, 6).astype(np.float32))
    hot = bell(rng, 6, 60000, "bf16")
    check(hot, u, temperature=np.full(6, 1000.0, np.float32), top_p=rng.uniform(0.1, 0.95, 6).astype(np.float32))


def test_infinities_and_nan():
    rng = np.random.default_rng(9)
    inf, nan = float("inf"), float("nan")
    for kind in ("bf16", "fp16", "fp32"):
        x = bell(rng, 7, 4000, kind)
        x[0, ::2] = -inf                # banned tokens
        x[1, 1:] = -inf                 # all but one
        x[2, :] = -inf
        x[3, 5:900] = nan
        x[4, :] = nan
        x[5, [17, 900, 3999]] = inf     # they share everything
        x[6, 0] = -inf
        x[6, 2500:] = -inf
        check(x, rng.random(7))
        check(x, rng.random(7), **controls(rng, 7))
        check(x, rng.random(7), temperature=np.zeros(7, np.float32))
        assert sample(x, 4000, torch.full((7,), 0.9, device="cuda"))[0].tolist()[2] == -1


def test_shares_are_drawn_as_often_as_they_weigh():
    """20,000 evenly spaced numbers over one row: each token's count is its share of them, to one."""
    rng = np.random.default_rng(10)
    x = bell(rng, 1, 300, "fp32", std=1.0, peaks=1)
    many = 20000
    u = (torch.arange(many, device="cuda") + 0.5) / many
    token, _ = sample(x.expand(many, 300).contiguous(), 300, u)
    share = torch.softmax(x[0].double(), 0) * many
    count = torch.bincount(token[:many].long(), minlength=300).double()
    assert float((count - share).abs().max()) <= 1.01


def test_the_result_depends_on_the_row_alone():
    """The same row among others, alone, at another alignment and again: the same token and probability."""
    rng = np.random.default_rng(11)
    x, u = bell(rng, 150, 30011, "bf16"), rng.random(150)
    c = controls(rng, 150, top_k=0)
    token, prob = check(x, u, **c)
    for r in (0, 1, 77, 149):
        one, share = check(x[r:r + 1], u[r:r + 1], **{k: v[r:r + 1] for k, v in c.items()})
        assert one[0] == token[r] and share[0] == prob[r]
    again, shares = check(x, u, **c)
    assert torch.equal(again, token) and torch.equal(shares, prob)


def test_replayed_graph_and_another_stream():
    rng = np.random.default_rng(12)
    x = bell(rng, 3, 107520, "bf16")
    u = torch.zeros(3, device="cuda")
    p = torch.full((3,), 0.9, device="cuda")
    work = torch.empty(max(16, lib().plamo_kernel_sample_workspace(3, 107520)), dtype=torch.uint8, device="cuda")
    sample(x, 107520, u, top_p=p, workspace=work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token, prob = sample(x, 107520, u, top_p=p, workspace=work)
    s = torch.cuda.Stream()
    for turn in range(4):
        x.copy_(bell(rng, 3, 107520, "bf16"))
        u.copy_(torch.from_numpy(rng.random(3)))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        eager, share = check(x, u.cpu().numpy(), top_p=np.full(3, 0.9, np.float32))
        assert torch.equal(token[:3], eager) and torch.equal(prob[:3], share)


@pytest.mark.parametrize("temperature", [1e-3, 1e-6, 1e-10, 3e-13, 1e-14, 2.2e-15, 1e-20, 1e-38])
def test_temperatures_near_zero(temperature):
    """Neighbouring logits are any number of the weights' steps apart; some share the largest."""
    rng = np.random.default_rng(13)
    for kind in ("bf16", "fp32"):
        x = bell(rng, 4, 20000, kind)
        top = x.amax(1)
        x[0, 5] = x[0, 19000] = top[0]
        x[1, 7] = torch.nextafter(top[1].float(), torch.tensor(-1.0, device="cuda"))
        x[2] = torch.nextafter(top[2].float(), torch.tensor(-1.0, device="cuda"))
        x[2, 11] = top[2]
        check(x, rng.random(4), temperature=np.full(4, temperature, np.float32))
        check(x, rng.random(4), temperature=np.full(4, temperature, np.float32), top_p=np.full(4, 0.5, np.float32))


def test_borders_among_negative_logits():
    """Packed pairs are looked over before they are taken apart: neighbours of every kind beside a border."""
    rng = np.random.default_rng(14)
    for kind in ("bf16", "fp16", "fp32"):
        x = -(rng.random((12, 40001)) * 30 + 2)
        x[:, 1::2] = -200 - rng.random((12, 20000))      # upper halves far lower than lower ones
        x[6:] = x[6:][:, ::-1]
        for r in range(12):
            few = rng.integers(0, 40001, 90)
            x[r, few] = -1.5 - rng.random(90) * 0.1
            x[r, few + (few < 40000)] = rng.choice([-np.inf, np.nan, -1.53, -0.0 - 3, 1e-30])
        x = torch.from_numpy(x.copy()).to(TYPES[kind]).cuda()
        check(x, rng.random(12), top_k=rng.integers(1, 90, 12).astype(np.int32))
        check(x, rng.random(12), top_p=rng.uniform(0.3, 0.999, 12).astype(np.float32))
        inf = x.clone()
        inf[:, ::7] = float("nan")
        inf[:, 35001] = float("inf")
        check(inf, rng.random(12), top_k=rng.integers(1, 90, 12).astype(np.int32))
        raw = {2: (torch.int16, 0x7F81 if kind == "bf16" else 0x7C01), 4: (torch.int32, 0x7F800001)}[x.element_size()]
        x.view(raw[0])[:, 3::5] = raw[1]                 # signalling NaN
        assert torch.isnan(x[:, 3::5]).all()
        check(x, rng.random(12), top_k=rng.integers(1, 90, 12).astype(np.int32))
        check(x, rng.random(12), top_p=rng.uniform(0.3, 0.999, 12).astype(np.float32))
        check(x, rng.random(12), temperature=np.zeros(12, np.float32))
    alone = torch.full((2, 20000), float("nan"), dtype=torch.bfloat16, device="cuda")
    alone[0, 12345] = float("inf")
    alone[1, 12346] = -7.0
    check(alone, [0.5, 0.5])
    check(alone, [0.5, 0.5], top_k=np.full(2, 3, np.int32))


def test_many_rows_beyond_the_lists():
    """Hundreds of rows whose kept tokens no list holds, among others whose it does."""
    rng = np.random.default_rng(15)
    x = bell(rng, 300, 9001, "bf16")
    k = rng.integers(1, 9001, 300).astype(np.int32)
    k[::3] = rng.integers(1, 60, 100)
    check(x, rng.random(300), top_k=k)
    check(x, rng.random(300), top_k=k, top_p=rng.uniform(0.1, 0.99, 300).astype(np.float32),
          temperature=np.where(rng.random(300) < 0.2, 0, 3.0).astype(np.float32))


def test_calls_on_two_streams_with_their_own_workspaces():
    rng = np.random.default_rng(16)
    cases = []
    for rows, n in ((5, 107520), (64, 30011), (1, 700)):
        x, u, c = bell(rng, rows, n, "bf16"), rng.random(rows).astype(np.float32), controls(rng, rows)
        want = check(x, u, **c)
        put = {k: torch.from_numpy(v).cuda() for k, v in c.items()}
        work = torch.full((max(16, lib().plamo_kernel_sample_workspace(rows, n)),), 0xFF, dtype=torch.uint8, device="cuda")
        cases.append((x, n, torch.from_numpy(u).cuda(), put, work, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for x, n, u, put, work, want, s in cases:
            with torch.cuda.stream(s):
                got.append((sample(x, n, u, workspace=work, **put), want, x.shape[0]))
    torch.cuda.synchronize()
    for (token, prob), want, rows in got:
        assert torch.equal(token[:rows], want[0]) and torch.equal(prob[:rows], want[1])


@pytest.mark.parametrize("n", [1, 5, 64, 1000, 4097, 9001])
def test_short_rows_in_more_than_all_workgroups(n):
    """The same rows among few and among many: short ones are drawn from by one workgroup or in several steps."""
    rng = np.random.default_rng([17, n])
    for kind in ("bf16", "fp32"):
        wide = torch.full((300, n + 1), 1e30, dtype=TYPES[kind], device="cuda")
        wide[:, :n] = bell(rng, 300, n, kind)
        x, u, c = wide[:, :n], rng.random(300), controls(rng, 300)
        token, prob = check(x, u, **c)
        few, share = check(x[100:140], u[100:140], **{k: v[100:140] for k, v in c.items()})
        assert torch.equal(few, token[100:140]) and torch.equal(share, prob[100:140])
        check(x, u)


def test_more_rows_than_a_grid_has_in_other_directions():
    rows = 70000
    x = torch.zeros(rows, 3, dtype=torch.bfloat16, device="cuda")
    x[torch.arange(rows), torch.arange(rows) % 3] = 5
    u = torch.full((rows,), 0.5, device="cuda")
    work = torch.empty(lib().plamo_kernel_sample_workspace(rows, 3), dtype=torch.uint8, device="cuda")
    token, prob = sample(x, 3, u, workspace=work)
    assert torch.equal(token[:rows].long().cpu(), torch.arange(rows) % 3) and int(token[rows]) == -7


def test_infinite_temperature_draws_evenly():
    rng = np.random.default_rng(18)
    for rows, n in ((5, 700), (3, 40001), (300, 900)):
        x = bell(rng, rows, n, "bf16")
        x[:, ::5] = -float("inf")
        x[:, 3] = float("nan")
        for mix in ("none", "all", "top_p"):
            check(x, rng.random(rows), **controls(rng, rows, **MIXES[mix], temperature=np.inf))


def test_the_largest_finite_value_beside_infinity():
    rng = np.random.default_rng(19)
    for n in (900, 40001):
        x = torch.full((6, n), torch.finfo(torch.float32).max, device="cuda")
        x[:, 1::2] = -torch.finfo(torch.float32).max
        x[3:, [5, 800]] = float("inf")
        for c in ({}, {"top_k": 3}, {"top_p": 0.5}, {"min_p": 0.5}, {"temperature": 1e38}, {"temperature": 0.0}):
            check(x, rng.random(6), **{k: np.full(6, v, np.int32 if k == "top_k" else np.float32) for k, v in c.items()})


def test_many_equal_logits_in_a_list():
    """Lists of a few hundred to two thousand tokens of one, two and many logits, beside each list's length."""
    rng = np.random.default_rng(20)
    for n in (5000, 70000):
        for count in (255, 256, 257, 600, 2047, 2048, 2049):
            x = torch.full((4, n), -40.0, device="cuda")
            for r, parts in enumerate(([1.0], [1.0, 1.0078125], [1.0, 1.0000001, 1.25], rng.random(count))):
                at = torch.from_numpy(rng.permutation(n)[:count]).cuda()
                x[r, at] = torch.from_numpy(rng.choice(parts, count)).float().cuda()
            for kind in ("fp32", "bf16", "fp16"):
                check(x.to(TYPES[kind]), rng.random(4), top_k=np.full(4, min(count, 1000), np.int32))
                check(x.to(TYPES[kind]), rng.random(4), top_p=np.full(4, 0.7, np.float32))
                check(x.to(TYPES[kind]), rng.random(4))
