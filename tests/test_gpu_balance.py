"""The balance losses over the superpoints against the formulas in float64.

Tolerances, e = 2^-24.  Pairs form: a share is rounded once, its product with the scale once: 2 e relative on a gradient
(3 e where it is added to another, of both); the loss sums exact products of rounded terms in double: 3 e of the sum of
their magnitudes, and e for itself.  Table form, a row with R the range of its values and d the length of a thread's
column sum and the tree behind it: an exponential is 4 e + 2 R e off (the difference to the row's largest value and its
product with log2(e) are rounded to R e together, half of each), sums d e more, so `inner` = sum p share is
(2 R + d + 8) e sum p |share| off and a gradient k p (share - inner) is (2 R + d + 12) e k p (|share| + 2 sum p |share|)
off, plus half a unit of a 16-bit type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _indices(N, K, M, gen, outside=0.0):
    idx = (torch.rand(N, K, generator=gen) ** 2 * M).long().clamp_(max=M - 1)
    if outside:
        bad = torch.rand(N, K, generator=gen) < outside
        idx[bad] = torch.tensor([-1, M, -2 ** 40, 2 ** 33, M + 7])[torch.randint(0, 5, (int(bad.sum()),), generator=gen)]
    return idx


def _counts(idx, M, mask):
    on = (idx >= 0) & (idx < M)
    if mask is not None:
        on = on & mask[:, None]
    c = torch.bincount(idx[on], minlength=M) if bool(on.any()) else torch.zeros(M, dtype=torch.int64)
    return c, on, int(c.sum()), idx.shape[0] if mask is None else int(mask.sum())


PAIRS = [(1, 1, 1, None, 0.0), (7, 3, 8192, 0.2, 0.1), (100_001, 5, 8193, 0.2, 0.1), (1, 3, 512, None, 0.0), (1000, 3, 512, None, 0.0), (1001, 8, 7, 0.3, 0.1),
         (33, 5, 9000, 0.5, 0.2), (50_003, 3, 512, 0.02, 0.0), (20_000, 2, 70_000, 0.1, 0.1), (3000, 16, 65_535, None, 0.1),
         (257, 4, 100, 1.0, 0.0), (64, 2, 10, None, 1.0), (5, 40, 3, 0.2, 0.2), (300_000, 8, 4096, 0.3, 0.01)]


@pytest.mark.parametrize("N,K,M,masked,outside", PAIRS)
def test_pairs_vs_formula(N, K, M, masked, outside):
    from fsgs.loss import balance_loss, balance_value_and_grad
    gen = torch.Generator().manual_seed(N + K)
    idx = _indices(N, K, M, gen, outside)
    w = torch.softmax(2 * torch.randn(N, K, generator=gen), dim=1)
    mask = None if masked is None else torch.rand(N, generator=gen) >= masked
    c, on, T, n = _counts(idx, M, mask)
    share = torch.zeros(N, K, dtype=torch.float64)
    if T and n:
        share[on] = M * c.double()[idx[on]] / (T * n)
    terms = share * w.double()
    w[~on] = float("nan")                     # what does not count is not read into anything
    dev = [t.cuda() if t is not None else None for t in (w, idx, mask)]
    loss, grad, counts = balance_value_and_grad(dev[0], dev[1], M, mask=dev[2], weight=0.25)
    assert torch.equal(counts.cpu(), c) and counts.dtype == torch.int64
    assert abs(float(loss) - 0.25 * float(terms.sum())) <= 5 * E * 0.25 * float(terms.sum())
    assert bool(((grad.cpu().double() - 0.25 * share).abs() <= 2 * E * 0.25 * share).all())
    base = torch.randn(N, K, generator=gen)
    into = base.cuda()
    _, same, _ = balance_value_and_grad(dev[0], dev[1], M, mask=dev[2], weight=0.25, grad=into)
    assert same is into
    assert bool(((into.cpu().double() - (base.double() + 0.25 * share)).abs() <= 3 * E * (0.25 * share + base.abs())).all())
    leaf = dev[0].clone().requires_grad_()
    value, counts = balance_loss(leaf, dev[1], M, mask=dev[2])
    (3.0 * value).backward()
    assert torch.equal(counts.cpu(), c) and abs(float(value) - float(terms.sum())) <= 5 * E * float(terms.sum())
    assert bool(((leaf.grad.cpu().double() - 3.0 * share).abs() <= 3 * E * 3.0 * share).all())


def _table_reference(z, idx, mask):
    M = z.shape[1]
    c, _, T, n = _counts(idx, M, mask)
    z = z.double()
    p = torch.softmax(z, dim=1)
    p[(z == -math.inf).all(dim=1)] = 0.0
    if mask is not None:
        p[~mask] = 0.0
    if T == 0 or n == 0:
        return c, 0.0, torch.zeros_like(p), torch.zeros_like(p)
    f = M * c.double() / T / n
    grad = p * (f - (p @ f)[:, None])
    centred = (M * c.double() - T) / (T * n)
    spread = (p * centred.abs()).sum(dim=1, keepdim=True)
    fin = torch.where(torch.isfinite(z), z, z.new_tensor(0.0))
    R = (z.amax(dim=1, keepdim=True).clamp(min=-1e30) - torch.where(torch.isfinite(z), z, z.new_tensor(1e30)).amin(dim=1, keepdim=True)).clamp(0, 200)
    del fin
    return c, float((p @ f).sum()), grad, (2 * R + M / 32 + 16 + 12) * E * p * (centred.abs() + 2 * spread)


TABLES = [(1, 1, 1, None), (1, 1, 2, None), (5, 2, 3, 0.5), (100, 3, 128, None), (100, 3, 129, 0.3), (77, 2, 333, 0.1),
          (1000, 3, 512, None), (64, 4, 513, 0.2), (40, 8, 2048, None), (33, 2, 2049, 0.2), (20, 3, 8192, None),
          (10, 3, 8193, 0.2), (6, 2, 20_011, None), (3000, 3, 512, 1.0), (1003, 3, 8, 0.1), (333, 2, 64, None),
          (65, 2, 65, 0.2), (50, 3, 256, 0.1), (50, 3, 260, None), (30, 3, 1024, 0.1), (30, 3, 1025, None), (21, 2, 4096, None),
          (21, 2, 4100, 0.2), (9, 2, 8188, None)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K,M,masked", TABLES)
def test_table_vs_formula(N, K, M, masked, dtype):
    from fsgs.loss import table_balance_loss, table_balance_value_and_grad
    gen = torch.Generator().manual_seed(N * M)
    idx = _indices(N, K, M, gen, 0.05 if N > 50 else 0.0)
    z = (2 * torch.randn(N, M, generator=gen)).to(dtype)
    mask = None if masked is None else torch.rand(N, generator=gen) >= masked
    c, want, g64, tol = _table_reference(z, idx, mask)
    dz, di, dm = z.cuda(), idx.cuda(), None if mask is None else mask.cuda()
    loss, grad, counts = table_balance_value_and_grad(dz, di, mask=dm, weight=0.5)
    assert torch.equal(counts.cpu(), c) and grad.dtype == dtype and grad.shape == z.shape
    off = float(tol.sum()) + 4 * E * abs(want)
    assert abs(float(loss) - 0.5 * want) <= 0.5 * off, (float(loss), want)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-40
    close = lambda got, k: bool(((got.cpu().double() - k * g64).abs() <= k * tol + HALF[dtype] * (k * g64.abs() + k * tol) + tiny).all())  # noqa: E731
    assert close(grad, 0.5)
    leaf = dz.clone().requires_grad_()
    value, counts = table_balance_loss(leaf, di, mask=dm)
    (2.0 * value).backward()
    assert torch.equal(counts.cpu(), c) and abs(float(value) - want) <= off and close(leaf.grad, 2.0)


def test_table_rows_with_infinities_and_strides():
    """Columns at -infinity, rows of nothing else, masked rows full of NaN; a table that is a slice of a wider one, one
    with its rows apart, a transposed one."""
    from fsgs.loss import table_balance_loss, table_balance_value_and_grad
    gen = torch.Generator().manual_seed(3)
    N, M = 60, 70
    idx = _indices(N, 3, M, gen)
    z = torch.randn(N, M, generator=gen)
    z[:, 5] = -math.inf
    z[7] = -math.inf
    z[8, 1:] = -math.inf
    z[9] = torch.finfo(torch.float32).min        # a row of nothing but the type's lowest value: all alike
    mask = torch.ones(N, dtype=torch.bool)
    mask[11] = False
    c, want, g64, tol = _table_reference(z, idx, mask)
    z[11] = math.nan
    assert float(g64[7].abs().max()) == 0.0
    wide = torch.full((N, M + 9), math.nan)
    wide[:, 4:4 + M] = z
    tall = torch.full((2 * N, M), math.nan)
    tall[::2] = z
    for t in (z.cuda(), wide.cuda()[:, 4:4 + M], tall.cuda()[::2], z.t().contiguous().cuda().t()):
        loss, grad, counts = table_balance_value_and_grad(t, idx.cuda(), mask=mask.cuda())
        assert torch.equal(counts.cpu(), c)
        assert abs(float(loss) - want) <= float(tol.sum()) + 4 * E * want
        assert bool(((grad.cpu().double() - g64).abs() <= tol + 1e-40).all())
    z[20, 3] = math.nan                           # a NaN that counts reaches its row and the loss, and no other row
    loss, grad, _ = table_balance_value_and_grad(z.cuda(), idx.cuda(), mask=mask.cuda())
    assert math.isnan(float(loss)) and torch.isnan(grad).any(dim=1).nonzero().flatten().tolist() == [20]
    # nobody bound: no loss, no gradient
    loss, grad, counts = table_balance_value_and_grad(torch.randn(4, 9).cuda(), torch.full((4, 2), -1).cuda())
    assert float(loss) == 0.0 and not bool(grad.any()) and not bool(counts.any())
    leaf = torch.zeros(0, 9, device="cuda", requires_grad=True)
    value, counts = table_balance_loss(leaf, torch.zeros(0, 2, dtype=torch.int64, device="cuda"))
    value.backward()
    assert float(value) == 0.0 and leaf.grad.shape == (0, 9)


def test_gradients_against_differences():
    """Central differences of the loss itself.  L = M/(T n) sum p c with c <= T: along one table entry its third
    derivative is at most 6 M / n (that of a softmax probability is below 1, times c / T <= 1, six terms), so a step h is
    off by h^2 M / n, and by the rounding of two losses of at most M, 2 x 8 e M / (2 h)."""
    from fsgs.loss import balance_value_and_grad, table_balance_value_and_grad
    gen = torch.Generator().manual_seed(1)
    N, K, M, h = 5, 2, 6, 2.0 ** -6
    idx = _indices(N, K, M, gen).cuda()
    z, w = torch.randn(N, M, generator=gen).cuda(), torch.rand(N, K, generator=gen).cuda()
    _, gz, _ = table_balance_value_and_grad(z, idx)
    _, gw, _ = balance_value_and_grad(w, idx, M)
    tol = h * h * M / N + 8 * E * M / h
    for x, g, f in ((z, gz, lambda t: table_balance_value_and_grad(t, idx)[0]), (w, gw, lambda t: balance_value_and_grad(t, idx, M)[0])):
        for k in range(x.numel()):
            up, down = x.clone().view(-1), x.clone().view(-1)
            up[k] += h
            down[k] -= h
            d = (float(f(up.view_as(x))) - float(f(down.view_as(x)))) / (2 * h)
            assert abs(d - float(g.view(-1)[k])) <= tol, (k, d, float(g.view(-1)[k]))


def test_repeats_bit_for_bit_and_in_a_graph():
    from fsgs.loss import balance_value_and_grad, table_balance_value_and_grad
    gen = torch.Generator().manual_seed(2)
    N, K, M = 40_000, 3, 300
    idx, w = _indices(N, K, M, gen).cuda(), torch.rand(N, K, generator=gen).cuda()
    z = torch.randn(N, M, generator=gen).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for call in (lambda: balance_value_and_grad(w, idx, M), lambda: table_balance_value_and_grad(z, idx)):
            first, second = call(), call()
            assert all(torch.equal(a, b) for a, b in zip(first, second))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                held = call()
            old = idx.clone()
            for k in range(3):
                idx.copy_((old + 31 * k) % M)
                graph.replay()
                assert all(torch.equal(a, b) for a, b in zip(held, call()))
            idx.copy_(old)
    torch.cuda.current_stream().wait_stream(stream)


def test_refusals():
    from fsgs.loss import balance_loss, balance_value_and_grad, table_balance_loss
    w, idx = torch.ones(4, 2, device="cuda"), torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    ok = torch.ones(4, dtype=torch.bool, device="cuda")
    for call in (lambda: balance_loss(w.double(), idx, 3), lambda: balance_loss(w, idx.int(), 3), lambda: balance_loss(w, idx, 0),
                 lambda: balance_loss(w, idx[:3], 3), lambda: balance_loss(w[:, :1], idx, 3), lambda: balance_loss(w, idx.cpu(), 3),
                 lambda: balance_loss(w, idx, 3, mask=ok[:3]), lambda: balance_loss(w, idx, 3, mask=ok.float()),
                 lambda: balance_loss(w, idx, 3, mask=ok.cpu()), lambda: balance_loss(w[0], idx, 3),
                 lambda: balance_loss(torch.ones(4, 0, device="cuda"), idx[:, :0], 3),
                 lambda: balance_value_and_grad(w, idx, 3, grad=torch.zeros(2, 4, device="cuda").t()),
                 lambda: balance_value_and_grad(w, idx, 3, grad=torch.zeros(4, 2)),
                 lambda: table_balance_loss(w.double(), idx), lambda: table_balance_loss(w[0], idx),
                 lambda: table_balance_loss(torch.ones(4, 0, device="cuda"), idx), lambda: table_balance_loss(w, idx[:, 0])):
        with pytest.raises(RuntimeError):
            call()


def test_autograd_of_the_losses():
    """Through other operations on both sides, with an upstream factor on the device; no gradient asked for; the table
    changed between the passes; a second derivative."""
    from fsgs.loss import balance_loss, balance_value_and_grad, table_balance_loss, table_balance_value_and_grad
    gen = torch.Generator().manual_seed(6)
    N, K, M = 500, 3, 40
    idx = _indices(N, K, M, gen).cuda()
    raw, z = torch.randn(N, K, generator=gen).cuda(), torch.randn(N, M, generator=gen).cuda()
    a = raw.clone().requires_grad_()
    w = torch.softmax(a, dim=1)
    loss, counts = balance_loss(w, idx, M)
    assert not counts.requires_grad and loss.requires_grad
    (loss ** 2).backward()
    value, grad, _ = balance_value_and_grad(w, idx, M)
    assert not value.requires_grad and not grad.requires_grad and torch.equal(value, loss.detach())
    p = w.detach().double()
    up = 2 * value.double() * grad.double()
    want = p * (up - (p * up).sum(dim=1, keepdim=True))
    assert float((a.grad.double() - want).abs().max()) <= 16 * E * float((p * up.abs()).max())
    b = z.clone().requires_grad_()
    loss, _ = table_balance_loss(b * 1.0, idx)
    (3.0 * loss).backward()
    _, grad, _ = table_balance_value_and_grad(z, idx)
    assert float((b.grad - 3.0 * grad).abs().max()) <= 4 * E * 3.0 * float(grad.abs().max())
    with torch.no_grad():
        assert not table_balance_loss(b, idx)[0].requires_grad and not balance_loss(a, idx, M)[0].requires_grad
    c = (z.clone().requires_grad_() * 1.0)
    loss, _ = table_balance_loss(c, idx)
    with torch.no_grad():
        c += 1.0
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()
    d = z.clone().requires_grad_()
    loss, _ = table_balance_loss(d, idx)
    g, = torch.autograd.grad(loss ** 2, d, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


def test_pairs_at_odd_addresses():
    """Indices, weights and the gradient that is added to, each one element off an aligned start: the same results."""
    from fsgs.loss import balance_value_and_grad
    gen = torch.Generator().manual_seed(8)
    N, K, M = 3001, 3, 77
    idx, w = _indices(N, K, M, gen, 0.05).cuda(), torch.rand(N, K, generator=gen).cuda()
    mask = (torch.rand(N, generator=gen) > 0.2).cuda()
    loss, grad, counts = balance_value_and_grad(w, idx, M, mask=mask)
    odd = lambda t: torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
    into = odd(torch.ones_like(w))
    loss2, same, counts2 = balance_value_and_grad(odd(w), odd(idx), M, mask=odd(mask), grad=into)
    assert torch.equal(counts, counts2) and same is into
    assert abs(float(loss) - float(loss2)) <= 4 * E * float(loss)
    assert torch.equal(into, 1.0 + grad)


def test_tables_beyond_32_bits_of_elements():
    """600 k x 4000 bf16, 2.4e9 elements: the first and the last rows against the formula."""
    from fsgs.loss import table_balance_value_and_grad
    N, M = 600_000, 4000
    gen = torch.Generator("cuda").manual_seed(1)
    z = torch.empty(N, M, dtype=torch.bfloat16, device="cuda")
    z.normal_(generator=gen)
    idx = (torch.rand(N, 2, device="cuda", generator=gen) ** 2 * M).long().clamp_(max=M - 1)
    weight = 2.0 ** 20                      # brings the gradients into the range in which bf16 keeps its precision
    loss, grad, counts = table_balance_value_and_grad(z, idx, weight=weight)
    assert torch.equal(counts, torch.bincount(idx.reshape(-1), minlength=M))
    f = M * counts.double() / (2 * N) / N
    for rows in (slice(0, 50), slice(N - 50, N)):
        p = torch.softmax(z[rows].double(), dim=1)
        want = weight * p * (f - (p @ f)[:, None])
        centred = (M * counts.double() - 2 * N) / (2 * N) / N
        tol = weight * (2 * 12 + M / 32 + 28) * E * p * (centred.abs() + 2 * (p * centred.abs()).sum(dim=1, keepdim=True))
        assert bool(((grad[rows].double() - want).abs() <= tol + HALF[torch.bfloat16] * (want.abs() + tol)).all())
    assert math.isfinite(float(loss))


def test_a_captured_backward_pass():
    """Forward and backward of both losses in one graph, no other graph of the leaves alive; replayed with other inputs."""
    from fsgs.loss import balance_loss, balance_value_and_grad, table_balance_loss, table_balance_value_and_grad
    gen = torch.Generator().manual_seed(9)
    N, K, M = 700, 2, 40
    idx = _indices(N, K, M, gen).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        z, w = torch.randn(N, M, device="cuda").requires_grad_(), torch.rand(N, K, device="cuda").requires_grad_()

        def both():
            a, b = table_balance_loss(z, idx)[0], balance_loss(w, idx, M)[0]
            return torch.autograd.grad(a + b, (z, w))

        both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = both()
        for k in range(2):
            with torch.no_grad():
                z.copy_(torch.randn(N, M, device="cuda"))
            idx.copy_((idx + 7) % M)
            graph.replay()
            assert torch.equal(held[0], table_balance_value_and_grad(z, idx)[1])
            assert torch.equal(held[1], balance_value_and_grad(w, idx, M)[1])
    torch.cuda.current_stream().wait_stream(stream)


@pytest.mark.parametrize("of", ["pairs", "table"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_a_captured_backward_pass_beside_a_living_graph(of, accumulate):
    """A loss of the same leaf is held, made on another stream: refused, and the same capture goes on without the backward."""
    from fsgs.loss import balance_loss, balance_value_and_grad, table_balance_loss, table_balance_value_and_grad
    gen = torch.Generator().manual_seed(10)
    N, K, M = 300, 2, 20
    idx = _indices(N, K, M, gen).cuda()
    x = (torch.rand(N, K, generator=gen) if of == "pairs" else torch.randn(N, M, generator=gen)).cuda().requires_grad_()
    loss = (lambda: balance_loss(x, idx, M)[0]) if of == "pairs" else (lambda: table_balance_loss(x, idx)[0])
    values = (lambda: balance_value_and_grad(x, idx, M)) if of == "pairs" else (lambda: table_balance_value_and_grad(x, idx))
    held = loss()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        values()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = loss()
            with pytest.raises(RuntimeError, match="value_and_grad"):
                captured.backward() if accumulate else torch.autograd.grad(captured, x)
            out = values()
        graph.replay()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    want = values()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]) and torch.equal(captured.detach(), want[0])
    assert x.grad is None
    (grad,) = torch.autograd.grad(held, x)                          # the held graph works as before
    assert torch.equal(grad, want[1])
    del captured, held                                              # let go of: the same capture now holds its backward pass
    with torch.cuda.stream(stream):
        torch.autograd.grad(loss(), x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            (again,) = torch.autograd.grad(loss(), x)
        graph.replay()
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(again, want[1])


def test_the_gradient_added_to_counts_as_modified():
    from fsgs.loss import balance_value_and_grad
    into = torch.zeros(50, 2, device="cuda")
    factor = torch.ones(50, 2, device="cuda", requires_grad=True)
    loss = (factor * into).sum()                   # saves `into`
    version = into._version
    w, idx = torch.rand(50, 2, device="cuda"), torch.zeros(50, 2, dtype=torch.int64, device="cuda")
    balance_value_and_grad(w, idx, 5, grad=into)
    assert into._version > version and w._version == 0 and idx._version == 0
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()
    with torch.inference_mode():
        plain = torch.zeros(50, 2, device="cuda")
        balance_value_and_grad(w, idx, 5, grad=plain)
    assert torch.equal(plain, into)


@pytest.mark.parametrize("N", [1, 1024])
def test_the_loss_of_terms_that_round_the_same_way(N):
    """A term of 1 and seven of a little over half a unit behind it, all shares a power of two: added one after another in
    float32 every addition rounds up, 7 e in all.  Asked for are 3 e of the sum (a share, a product, one addition) and e for
    the loss itself."""
    from fsgs.loss import balance_loss, balance_value_and_grad
    for order in (slice(None), slice(None, None, -1)):
        w = torch.tensor([1.0] + [1.01 * E] * 7).expand(N, 8).contiguous()
        idx = torch.arange(8).expand(N, 8).contiguous()
        if order.step:
            w = w.flip(1)
        want = float(w.double().sum()) / N
        for loss in (balance_value_and_grad(w.cuda(), idx.cuda(), 8)[0], balance_loss(w.cuda(), idx.cuda(), 8)[0]):
            assert abs(float(loss) - want) <= 4 * E * want


def test_running_out_of_memory_is_torchs_error():
    """Seen as ``torch.cuda.OutOfMemoryError`` by who catches it to try a smaller call, and the next call works."""
    from fsgs.loss import balance_loss, balance_value_and_grad, table_balance_loss, table_balance_value_and_grad
    from fsgs.optim import grad_norm
    one = torch.zeros(1, 1, device="cuda")
    w, idx = one.expand(2 ** 27, 8), one.long().expand(2 ** 27, 8)       # 4 and 8 GB where they are laid out
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction(2 ** 30 / total)
    try:
        for call in (lambda: balance_value_and_grad(w, idx, 3), lambda: balance_loss(w.detach().requires_grad_(), idx, 3),
                     lambda: table_balance_loss(w, idx), lambda: table_balance_value_and_grad(w, idx), lambda: grad_norm([w])):
            with pytest.raises(torch.cuda.OutOfMemoryError):
                call()
        assert float(balance_value_and_grad(w[:4].contiguous() + 1, idx[:4].contiguous(), 1)[0]) == 8.0
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)


def test_balance_of_the_table_weighting():
    """``balance_loss`` on the weights that ``lbs_weights`` blends from a table: its gradient reaches the K entries of each
    row that are read, and no other; ``table_balance_loss`` acts on the whole row.  A weight is a softmax in float32 of
    values within 8 of each other (20 e), its adjoint two products and a difference of terms below p |up| (16 e more)."""
    from fsgs.loss import balance_loss, table_balance_loss
    from fsgs.scene import lbs_weights
    gen = torch.Generator().manual_seed(12)
    N, K, M = 400, 3, 30
    idx = torch.rand(N, M, generator=gen).argsort(dim=1)[:, :K].contiguous()
    table = torch.randn(N, M, generator=gen)
    leaf = table.double().requires_grad_()
    w = leaf.gather(1, idx).softmax(dim=1)
    c = torch.bincount(idx.reshape(-1), minlength=M).double()
    up = M * c[idx] / (N * K * N)
    (w * up).sum().backward()
    own = table.cuda().requires_grad_()
    loss, counts = balance_loss(lbs_weights(None, idx.cuda(), "table", table=own), idx.cuda(), M)
    loss.backward()
    want = float((w * up).sum())
    assert torch.equal(counts.cpu().double(), c) and abs(float(loss) - want) <= 24 * E * want
    room = torch.zeros(N, M, dtype=torch.float64).scatter_(1, idx, (w * up).detach().sum(dim=1, keepdim=True).expand(N, K))
    assert bool(((own.grad.cpu().double() - leaf.grad).abs() <= 36 * E * room).all())
    # what no weight reads changes the loss over the whole row only
    other = table.clone().scatter_(1, idx, -math.inf)
    moved = torch.where(other == -math.inf, table, other + 3.0).cuda()
    assert torch.equal(balance_loss(lbs_weights(None, idx.cuda(), "table", table=moved), idx.cuda(), M)[0], loss.detach())
    assert not torch.equal(table_balance_loss(moved, idx.cuda())[0], table_balance_loss(own, idx.cuda())[0].detach())


def test_the_counts_are_the_callers():
    """Summed over ranks or steps in place before the backward pass, as counts are: the gradient is of the counts that the
    loss was formed with."""
    from fsgs.loss import balance_loss, balance_value_and_grad, table_balance_loss, table_balance_value_and_grad
    gen = torch.Generator().manual_seed(13)
    N, K, M = 300, 3, 20
    idx = _indices(N, K, M, gen).cuda()
    w, z = torch.rand(N, K, generator=gen).cuda(), torch.randn(N, M, generator=gen).cuda()
    for x, form, plain in ((w, lambda t: balance_loss(t, idx, M), lambda t: balance_value_and_grad(t, idx, M)),
                           (z, lambda t: table_balance_loss(t, idx), lambda t: table_balance_value_and_grad(t, idx))):
        want, grad, counts = plain(x)
        for change in (lambda c: c.mul_(2), lambda c: c.data.zero_()):
            leaf = x.clone().requires_grad_()
            loss, own = form(leaf)
            assert torch.equal(own, counts)
            change(own)
            loss.backward()
            assert torch.equal(loss.detach(), want) and torch.equal(leaf.grad, grad)
