"""Routing, token rows sorted by expert and back: against plain loops and 64-bit formulas, refusals, streams, graphs, and a run of them
around the grouped GEMM."""
import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import nvfp4_gemm
from nvfp4_gemm import _C, TokenOrder, linear, route_tokens, sort_tokens, unsort_tokens

gpu = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
ALL_TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- refusals: on the host, before anything reaches a GPU ------------------------------------------------------------


def error_of(rc):
    assert rc == 1
    return _C.lib().nvfp4_last_error().decode()


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="logits is a 2-D"):
        route_tokens(torch.zeros(2, 8), 2)
    with pytest.raises(RuntimeError, match="x is a 2-D"):
        sort_tokens(torch.zeros(2, 8), torch.zeros(2, 1, dtype=torch.int64), 4)
    order = TokenOrder(torch.zeros(2, 1, dtype=torch.int64), torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        unsort_tokens(torch.zeros(4, 8), order)
    with pytest.raises(RuntimeError, match="rows of the order"):
        unsort_tokens(torch.zeros(5, 8), order)


@pytest.mark.parametrize("experts, k, scores, dtype, ld, text", [
    (0, 1, 0, 1, 8, "experts"), (1025, 1, 0, 1, 2000, "experts"), (8, 0, 0, 1, 8, "k (0)"), (8, 9, 0, 1, 8, "k (9)"),
    (64, 33, 0, 1, 64, "k (33)"), (8, 2, 2, 1, 8, "score function"), (8, 2, 0, 3, 8, "type code"), (8, 2, 0, 1, 7, "row stride")])
def test_routing_refuses_sizes(experts, k, scores, dtype, ld, text):
    lib = _C.lib()
    assert text in error_of(lib.nvfp4_route_tokens(16, ld, dtype, 4, experts, k, scores, 1, 16, 16, None))
    assert text in error_of(lib.nvfp4_route_tokens_backward(16, ld, dtype, 4, experts, k, scores, 1, 16, 16, 16, None))


def test_routing_refuses_pointers():
    lib = _C.lib()
    assert "null" in error_of(lib.nvfp4_route_tokens(None, 8, 1, 4, 8, 2, 0, 1, 16, 16, None))
    assert "aligned" in error_of(lib.nvfp4_route_tokens(18, 8, 1, 4, 8, 2, 0, 1, 16, 16, None))
    assert lib.nvfp4_route_tokens(None, 8, 1, 0, 8, 2, 0, 1, None, None, None) == 0      # no token: nothing to do


@pytest.mark.parametrize("tokens, k, hidden, experts, alignment, m, ld, text", [
    (4, 0, 8, 4, 16, 64, 8, "k=0"), (4, 1, 0, 4, 16, 64, 8, "hidden=0"), (-1, 1, 8, 4, 16, 64, 8, "tokens=-1"),
    (4, 1, 8, 0, 16, 64, 8, "experts"), (4, 1, 8, 1025, 16, 64, 8, "experts"), (4, 1, 8, 4, 0, 64, 8, "alignment"),
    (4, 1, 8, 4, 16, 48, 8, "M is 64"), (4, 1, 8, 4, 16, 64, 7, "row stride"), (1 << 30, 2, 8, 4, 16, 64, 8, "too many"),
    ((1 << 31) - 40000, 1, 8, 1024, 1 << 20, 1 << 31, 8, "number of rows")])
def test_sorting_refuses_sizes(tokens, k, hidden, experts, alignment, m, ld, text):
    assert text in error_of(_C.lib().nvfp4_sort_tokens(16, ld, 0, tokens, k, hidden, 16, experts, alignment, m, 16, 16, 16, 16, None))


def test_sorting_and_its_gradients_refuse_pointers():
    lib = _C.lib()
    assert "null" in error_of(lib.nvfp4_sort_tokens(16, 8, 0, 4, 1, 8, None, 4, 16, 64, 16, 16, 16, 16, None))
    assert "aligned" in error_of(lib.nvfp4_sort_tokens(17, 8, 0, 4, 1, 8, 16, 4, 16, 64, 16, 16, 16, 16, None))
    assert "null" in error_of(lib.nvfp4_unsort_tokens(16, 8, 0, 64, None, None, 4, 1, 8, 16, None))
    assert "type code" in error_of(lib.nvfp4_unsort_tokens(16, 8, 7, 64, 16, None, 4, 1, 8, 16, None))
    assert "needs the rows" in error_of(lib.nvfp4_unsort_tokens_backward(16, 8, None, 8, 0, 64, 16, 16, 16, 4, 1, 8, 16, 16, None))
    assert "sources" in error_of(lib.nvfp4_unsort_tokens_backward(16, 8, 16, 8, 0, 64, 16, None, 16, 4, 1, 8, 16, 16, None))
    assert lib.nvfp4_unsort_tokens_backward(16, 8, 16, 8, 0, 64, 16, 16, 16, 4, 1, 8, None, None, None) == 0


@pytest.mark.parametrize("pairs, experts, alignment", [(0, 4, 16), (1, 4, 128), (7, 4, 16), (128, 128, 32), (1000, 3, 64), (33, 1, 1)])
def test_the_rows_of_the_buffer_bound_every_routing(pairs, experts, alignment):
    m = _C.sorted_rows(pairs, experts, alignment)
    assert m % alignment == 0
    # the worst routing: one pair in every group but one
    live = min(experts, pairs)
    sizes = [1] * (live - 1) + [pairs - live + 1] if live else []
    assert sum(-(-s // alignment) * alignment for s in sizes) <= m <= pairs + live * (alignment - 1)


# ---- routing ---------------------------------------------------------------------------------------------------------


def route_in_64_bits(logits, k, scores, renormalize):
    """(ids, weights) by a stable sort and the definitions; differentiable in `logits` (float64, host)."""
    order = torch.sort(logits.detach(), dim=1, descending=True, stable=True)[1][:, :k]
    top = logits.gather(1, order)
    live = top > -math.inf
    ids = torch.where(live, order, -1)
    log_s = torch.log_softmax(logits, dim=1) if scores == "softmax" else torch.nn.functional.logsigmoid(logits)
    chosen = log_s.gather(1, order)
    if renormalize:
        chosen = chosen - torch.logsumexp(chosen.masked_fill(~live, -math.inf), dim=1, keepdim=True)
    return ids, torch.where(live, torch.exp(chosen), 0.0)


def weight_bound(logits, k):
    """Relative error of an FP32 weight: exp(l - max) carries the rounding of its argument, |l - max| 2^-24, as do the terms of the sum it
    is divided by; expf is off by at most 2 steps, i.e. 2^-22, twice; the sum of E terms in a tree of log2 E + E / 32 additions and the
    division round once each.  Counted with every rounding at its largest."""
    finite = logits[torch.isfinite(logits)]
    spread = float(finite.max() - finite.min()) if finite.numel() else 0.0
    return (2 * max(spread, 1.0) + 16 + 5 + logits.shape[1] / 32 + 2) * 2.0 ** -24


@gpu
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens, experts, k", [(1, 1, 1), (3, 5, 5), (9, 32, 32), (17, 33, 2), (8, 64, 6), (65, 128, 8), (5, 200, 10), (40, 257, 4),
                                                (7, 512, 8), (6, 1000, 32), (3, 1024, 1)])
def test_routing_against_the_definitions(tokens, experts, k, scores, renormalize):
    for dtype in ALL_TYPES:
        logits = (torch.randn(tokens, experts, generator=gen(tokens * experts + k)) * 2).to(dtype)       # 16-bit logits tie
        ids, weights = route_tokens(logits.cuda(), k, scores=scores, renormalize=renormalize)
        want_ids, want = route_in_64_bits(logits.double(), k, scores, renormalize)
        assert ids.dtype == torch.int64 and weights.dtype == torch.float32
        assert torch.equal(ids.cpu(), want_ids)
        bound = weight_bound(logits.double(), k)
        assert (weights.cpu().double() - want).abs().le(bound * want).all()


@gpu
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_routing_gradient_against_the_definitions(scores, renormalize):
    for tokens, experts, k in ((1, 1, 1), (9, 33, 5), (64, 128, 8), (5, 1000, 32)):
        for dtype in ALL_TYPES:
            logits = (torch.randn(tokens, experts, generator=gen(experts)) * 2).to(dtype)
            logits[0, experts // 2] = -math.inf
            if tokens > 4:
                logits[3] = -math.inf                                     # nothing to route to
                logits[4, 2:] = -math.inf                                 # fewer experts than choices
            grad = torch.randn(tokens, k, generator=gen(k))
            leaf = logits.cuda().requires_grad_()
            ids, weights = route_tokens(leaf, k, scores=scores, renormalize=renormalize)
            got = torch.autograd.grad(weights, leaf, grad.cuda())[0]
            assert got.dtype == dtype
            exact = logits.double()
            exact[~torch.isfinite(exact)] = -1e4                          # as good as masked in 64 bits: exp underflows to 0
            exact.requires_grad_()
            want_ids, want_w = route_in_64_bits(exact, k, scores, renormalize)
            masked = ~torch.isfinite(logits.gather(1, want_ids))
            want = torch.autograd.grad(want_w, exact, grad.double().masked_fill(masked, 0.0))[0]
            want[~torch.isfinite(logits)] = 0.0
            assert torch.equal(ids.cpu(), want_ids.masked_fill(masked, -1))
            if tokens > 4:                                                # the row of -1e4 is no routing in 64 bits: zero by definition
                assert (ids[3] == -1).all() and (weights[3] == 0).all()
                want[3] = 0.0
            # the weights' bound on products of two scores and differences of gradients, then one rounding
            scale = 2 * grad.abs().max()
            tolerance = 4 * weight_bound(logits.double(), k) * scale + HALF_STEP[dtype] * want.abs() + 2.0 ** -25
            assert (got.cpu().double() - want).abs().le(tolerance).all(), (tokens, experts, dtype)


@gpu
def test_routing_gradient_against_differences():
    logits = torch.randn(4, 12, generator=gen(3), dtype=torch.float64)
    grad = torch.randn(4, 3, generator=gen(4), dtype=torch.float64)
    for scores in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            leaf = logits.float().cuda().requires_grad_()
            _, w = route_tokens(leaf, 3, scores=scores, renormalize=renormalize)
            got = torch.autograd.grad(w, leaf, grad.float().cuda())[0].cpu().double()
            h = 1e-5
            base = leaf.detach().cpu().double()
            for i in range(4):
                for j in range(12):
                    up, down = base.clone(), base.clone()
                    up[i, j] += h
                    down[i, j] -= h
                    slope = ((route_in_64_bits(up, 3, scores, renormalize)[1] - route_in_64_bits(down, 3, scores, renormalize)[1]) * grad).sum() / (2 * h)
                    assert abs(float(slope) - float(got[i, j])) < 1e-5    # h^2 and FP32 roundings of values below 10


@gpu
def test_routing_ties_masks_and_extremes():
    inf, low = math.inf, torch.finfo(torch.float32).min
    logits = torch.tensor([[1.0, 1.0, 1.0, 1.0], [0.0, -0.0, 0.0, -0.0], [-inf, 2.0, -inf, 1.0], [-inf] * 4, [low, low, -inf, low],
                           [low, 0.0, low, -inf], [1e30, -1e30, 3e38, 0.0], [-200.0, -210.0, -inf, -200.0]])
    want_ids = [[0, 1, 2], [0, 1, 2], [1, 3, -1], [-1, -1, -1], [0, 1, 3], [1, 0, 2], [2, 0, 3], [0, 3, 1]]
    for scores in ("softmax", "sigmoid"):
        ids, w = route_tokens(logits.cuda(), 3, scores=scores)
        assert ids.tolist() == want_ids
        third = torch.full((3,), 1 / 3)
        w = w.cpu()
        for row in (0, 1, 4):
            assert torch.allclose(w[row], third, rtol=1e-6, atol=0)
        assert (w[3] == 0).all() and w[2, 2] == 0 and torch.isfinite(w).all()
        # far below zero a sigmoid is exp: the same ratios as the softmax's, although every score underflows
        assert torch.allclose(w[7, :2], torch.tensor([0.5, 0.5]) / (1 + 0.5 * math.exp(-10)), rtol=1e-5, atol=0)
    nan = torch.tensor([[0.0, math.nan, 1.0], [0.0, inf, 1.0], [0.0, 2.0, 1.0]])
    ids, w = route_tokens(nan.cuda(), 2)
    assert ids.tolist() == [[1, 2], [1, 2], [1, 2]] and torch.isnan(w[0]).all() and torch.isnan(w[1]).all() and torch.isfinite(w[2]).all()


@gpu
def test_routing_takes_strided_logits_and_no_tokens():
    wide = torch.randn(10, 300, generator=gen(1)).cuda()
    part = wide[1::2, 7:107]
    ids, w = route_tokens(part, 4)
    again, w2 = route_tokens(part.contiguous(), 4)
    assert torch.equal(ids, again) and torch.equal(w, w2)
    ids, w = route_tokens(wide[:0], 4)
    assert ids.shape == w.shape == (0, 4)
    with pytest.raises(RuntimeError, match="contiguous along"):
        route_tokens(wide.t(), 4)
    with pytest.raises(RuntimeError, match="2-D"):
        route_tokens(wide.long(), 4)
    with pytest.raises(RuntimeError, match="scores"):
        route_tokens(wide, 4, scores="tanh")
    with pytest.raises(RuntimeError, match="overlap"):
        route_tokens(wide[:1].expand(4, 300), 4)


# ---- sorting ---------------------------------------------------------------------------------------------------------


def order_by_loops(ids, experts, alignment):
    flat = ids.reshape(-1).tolist()
    n, live = len(flat), min(experts, len(flat))
    m = (n + live * (alignment - 1)) // alignment * alignment
    place, source, m_indices, at = [-1] * n, [-1] * m, [-1] * m, 0
    groups = {}
    for p, e in enumerate(flat):
        groups.setdefault(e, []).append(p)
    for e in range(experts):
        pairs = groups.get(e, [])
        for i, p in enumerate(pairs):
            place[p], source[at + i] = at + i, p
        end = at + -(-len(pairs) // alignment) * alignment
        m_indices[at:end] = [e] * (end - at)
        at = end
    return torch.tensor(place, dtype=torch.int64).reshape(ids.shape), torch.tensor(source, dtype=torch.int32), torch.tensor(m_indices, dtype=torch.int32)


def some_ids(tokens, k, experts, seed, kind):
    g = gen(seed)
    if kind == "one":
        return torch.full((tokens, k), experts - 1, dtype=torch.int64)
    ids = torch.randint(0, experts, (tokens, k), generator=g)             # the same expert may come twice in a row
    if kind == "skewed":
        ids = torch.minimum(ids, torch.randint(0, experts, (tokens, k), generator=g)) // 2
    if kind == "holes":
        ids[torch.rand(tokens, k, generator=g) < 0.3] = -1
        ids[torch.rand(tokens, k, generator=g) < 0.1] = experts + 5
        ids[0] = -(1 << 40)
    return ids


SORT_SIZES = [(1, 1, 1, 8, 16), (1, 8, 128, 64, 128), (5, 3, 7, 13, 1), (16, 8, 128, 4096, 32), (33, 2, 1000, 24, 16), (513, 8, 64, 40, 128),
              (512, 8, 1024, 8, 16), (1100, 4, 16, 72, 64), (4099, 6, 64, 96, 128), (9001, 10, 1024, 16, 16), (70001, 3, 33, 8, 48)]


@gpu
@pytest.mark.parametrize("kind", ["uniform", "skewed", "holes", "one"])
@pytest.mark.parametrize("tokens, k, experts, hidden, alignment", SORT_SIZES)
def test_sorted_rows_are_where_the_loops_put_them(tokens, k, experts, hidden, alignment, kind):
    ids = some_ids(tokens, k, experts, tokens + k, kind)
    place, source, m_indices = order_by_loops(ids, experts, alignment)
    for dtype in ALL_TYPES:
        x = torch.randn(tokens, hidden, generator=gen(hidden)).to(dtype)
        rows, order = sort_tokens(x.cuda(), ids.cuda(), experts, alignment=alignment)
        assert torch.equal(order.place.cpu(), place) and torch.equal(order.source.cpu(), source) and torch.equal(order.m_indices.cpu(), m_indices)
        want = torch.zeros(len(source), hidden, dtype=dtype)
        want[source >= 0] = x[source[source >= 0].long() // k]
        assert rows.dtype == dtype and torch.equal(rows.cpu(), want)


@gpu
@pytest.mark.parametrize("hidden, offset, stride", [(1, 0, 1), (7, 0, 7), (8, 1, 24), (64, 2, 80), (64, 8, 72), (130, 0, 130), (1030, 3, 1040)])
def test_rows_of_any_width_and_alignment_move_whole(hidden, offset, stride):
    for tokens in (6, 1500):                                              # one kernel, three kernels
        ids = some_ids(tokens, 4, 9, 1, "holes")
        place, source, _ = order_by_loops(ids, 9, 16)
        for dtype in ALL_TYPES:
            base = torch.randn(tokens * stride + offset + hidden, generator=gen(2)).to(dtype).cuda()
            x = base.as_strided((tokens, hidden), (stride, 1), offset)
            rows, order = sort_tokens(x, ids.cuda(), 9, alignment=16)
            want = torch.zeros(len(source), hidden, dtype=dtype)
            want[source >= 0] = x.cpu()[source[source >= 0].long() // 4]
            assert torch.equal(rows.cpu(), want)
            # and back: rows with a stride of their own
            wide = torch.full((len(source), stride + 8), float("nan"), dtype=dtype, device="cuda")
            view = wide.as_strided((len(source), hidden), (stride + 8, 1), min(offset, 8))
            view.copy_(rows)
            w = torch.rand(tokens, 4, generator=gen(5))
            got = unsort_tokens(view, order, w.cuda())
            exact = sum_by_loops(want, place, w)
            assert (got.cpu().double() - exact).abs().le(sum_bound(want, place, w, dtype)).all()


@gpu
def test_sorting_nothing():
    rows, order = sort_tokens(torch.empty(0, 16, device="cuda"), torch.empty(0, 4, dtype=torch.int64, device="cuda"), 8)
    assert rows.shape == (0, 16) and order.place.shape == (0, 4) and order.source.shape == order.m_indices.shape == (0,)
    assert unsort_tokens(rows, order, torch.empty(0, 4, device="cuda")).shape == (0, 16)


# ---- and back --------------------------------------------------------------------------------------------------------


def sum_by_loops(rows, place, w):
    """sum_j w[t, j] * rows[place[t, j]] in 64 bits."""
    picked = torch.where(place[..., None] >= 0, rows.double()[place.clamp(min=0)], 0.0)
    return (picked * (w.double()[..., None] if w is not None else 1.0)).sum(dim=1)


def sum_bound(rows, place, w, dtype):
    """k products and additions in FP32 (FMA: one rounding each, of partial sums no larger than the sum of magnitudes), then one rounding."""
    picked = torch.where(place[..., None] >= 0, rows.double()[place.clamp(min=0)], 0.0).abs()
    size = (picked * (w.double().abs()[..., None] if w is not None else 1.0)).sum(dim=1)
    return size * (place.shape[1] * 2.0 ** -24 + 1.01 * HALF_STEP[dtype]) + (2.0 ** -25 if dtype == torch.float16 else 1e-40)


@gpu
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("tokens, k, experts, hidden, alignment", [(1, 1, 1, 8, 16), (3, 8, 16, 4096, 32), (7, 33, 40, 72, 16), (300, 6, 64, 520, 128),
                                                                   (2000, 2, 5, 24, 64)])
def test_rows_back_and_their_gradients(tokens, k, experts, hidden, alignment, weighted):
    for kind in ("uniform", "holes"):
        ids = some_ids(tokens, k, experts, 11, kind)
        place, source, m_indices = order_by_loops(ids, experts, alignment)
        order = TokenOrder(place.cuda(), source.cuda(), m_indices.cuda())
        m = len(source)
        for dtype in ALL_TYPES:
            rows = torch.randn(m, hidden, generator=gen(1)).to(dtype)
            rows[source < 0] = float("nan")                               # padding: nothing of it may be read
            w = torch.randn(tokens, k, generator=gen(2)) if weighted else None
            dy = torch.randn(tokens, hidden, generator=gen(3)).to(dtype)
            leaf = rows.cuda().requires_grad_()
            w_leaf = w.cuda().requires_grad_() if weighted else None
            y = unsort_tokens(leaf, order, w_leaf)
            clean = torch.where(source[:, None] >= 0, rows, torch.zeros((), dtype=dtype))
            assert y.dtype == dtype
            assert (y.detach().cpu().double() - sum_by_loops(clean, place, w)).abs().le(sum_bound(clean, place, w, dtype)).all()
            grads = torch.autograd.grad(y, [leaf] + ([w_leaf] if weighted else []), dy.cuda())
            pair = source.clamp(min=0).long()
            scale = w.reshape(-1)[pair] if weighted else torch.ones(m)
            want = torch.where(source[:, None] >= 0, dy.double()[pair // k] * scale.double()[:, None], 0.0)
            error = (grads[0].cpu().double() - want).abs()
            assert error.le(want.abs() * (1.01 * HALF_STEP[dtype] + 2.0 ** -24) + (2.0 ** -25 if dtype == torch.float16 else 1e-40)).all()
            assert (grads[0][source.cuda() < 0] == 0).all()
            if weighted:
                picked = torch.where(place[..., None] >= 0, clean.double()[place.clamp(min=0)], 0.0)
                terms = picked * dy.double()[:, None, :]
                # `hidden` FP32 multiply-adds, in chains of hidden / 256 and a tree over the block: counted as one chain
                assert (grads[1].cpu().double() - terms.sum(dim=2)).abs().le(terms.abs().sum(dim=2) * (hidden + 16) * 2.0 ** -24 + 1e-40).all()


@gpu
def test_gradients_that_are_wanted_alone():
    ids = some_ids(40, 4, 8, 3, "holes").cuda()
    x = torch.randn(40, 64, generator=gen(1)).cuda().requires_grad_()
    rows, order = sort_tokens(x, ids, 8, alignment=16)
    w = torch.rand(40, 4, generator=gen(2)).cuda().requires_grad_()
    both = torch.autograd.grad(unsort_tokens(rows, order, w).sum(), [rows, w], retain_graph=True)
    (only_rows,) = torch.autograd.grad(unsort_tokens(rows, order, w.detach()).sum(), [rows], retain_graph=True)
    (only_w,) = torch.autograd.grad(unsort_tokens(rows.detach(), order, w).sum(), [w])
    assert torch.equal(both[0], only_rows) and torch.equal(both[1], only_w)
    # through both: sum_j w_j over the pairs that have a row
    (dx,) = torch.autograd.grad(unsort_tokens(rows, order, w.detach()).sum(), [x])
    live = (w.detach() * (order.place >= 0)).double().sum(dim=1, keepdim=True).expand(40, 64)
    assert (dx.double() - live).abs().max() < 8 * 2.0 ** -22              # four products and four sums below 4


@gpu
def test_sort_gradient_is_the_sum_over_a_tokens_rows():
    for dtype in ALL_TYPES:
        for tokens, k, experts, hidden in ((9, 3, 5, 33), (700, 8, 64, 264)):
            ids = some_ids(tokens, k, experts, 21, "holes")
            place, source, _ = order_by_loops(ids, experts, 32)
            x = torch.randn(tokens, hidden, generator=gen(1)).to(dtype).cuda().requires_grad_()
            rows, order = sort_tokens(x, ids.cuda(), experts, alignment=32)
            g = torch.randn(len(source), hidden, generator=gen(2)).to(dtype)
            (dx,) = torch.autograd.grad(rows, x, g.cuda())
            assert dx.dtype == dtype
            assert (dx.cpu().double() - sum_by_loops(g, place, None)).abs().le(sum_bound(g, place, None, dtype)).all()
            rows, _ = sort_tokens(x, ids.cuda(), experts, alignment=32)
            (ones,) = torch.autograd.grad(rows.sum(), x)                  # a gradient that is one value, expanded
            assert torch.equal(ones.cpu().float(), (place >= 0).sum(dim=1, keepdim=True).float().expand(tokens, hidden))


@gpu
def test_places_outside_the_rows_are_not_read():
    rows = torch.randn(32, 16, generator=gen(1)).cuda()
    place = torch.tensor([[0, 32], [1 << 40, 5], [-7, -(1 << 50)]], device="cuda")
    order = TokenOrder(place, torch.full((32,), -1, dtype=torch.int32, device="cuda"), torch.zeros(32, dtype=torch.int32, device="cuda"))
    y = unsort_tokens(rows, order, torch.ones(3, 2, device="cuda"))
    assert torch.equal(y[0], rows[0]) and torch.equal(y[1], rows[5]) and (y[2] == 0).all()


@gpu
def test_offsets_beyond_32_bits():
    """More elements in the sorted buffer than 32 bits count: forward and backward, checked on the device."""
    tokens, k, experts, hidden = 66000, 8, 16, 8192
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randint(-8, 8, (tokens, hidden), generator=g, device="cuda").to(torch.bfloat16).requires_grad_()
    ids = torch.randint(0, experts, (tokens, k), generator=g, device="cuda")
    rows, order = sort_tokens(x, ids, experts, alignment=16)
    assert rows.numel() > 1 << 32
    assert (order.place >= 0).all() and order.place.max() > (1 << 32) // hidden
    for lo in range(0, tokens, 4096):
        assert torch.equal(rows.detach()[order.place[lo:lo + 4096]], x.detach()[lo:lo + 4096, None].expand(-1, k, -1))
    assert (rows.detach()[order.source < 0] == 0).all()
    w = torch.randint(1, 4, (tokens, k), generator=g, device="cuda").float().requires_grad_()
    y = unsort_tokens(rows, order, w)                                     # small whole numbers: exact in FP32, rounded once
    assert torch.equal(y.detach(), (x.detach().float() * w.detach().sum(dim=1, keepdim=True)).to(torch.bfloat16))
    dy = torch.zeros(tokens, hidden, dtype=torch.bfloat16, device="cuda")
    dy[:, ::97] = 1
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert torch.equal(dx.float(), dy.float() * w.detach().sum(dim=1, keepdim=True))
    assert torch.equal(dw, (x.detach()[:, ::97].float().sum(dim=1, keepdim=True)).expand(-1, k))


FIRST_CALL_IN_A_CAPTURE = """
import torch, nvfp4_gemm
from nvfp4_gemm import linear, route_tokens, sort_tokens, unsort_tokens
x = torch.randn(600, 64, device="cuda").to(torch.bfloat16)
gate = torch.randn(16, 64, device="cuda").to(torch.bfloat16)
torch.cuda.synchronize()
def step():
    ids, w = route_tokens(linear(x, gate, out_dtype=torch.float32), 4)
    rows, order = sort_tokens(x, ids, 16)
    return unsort_tokens(rows, order, w)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = step()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, step())
"""


@gpu
def test_the_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys

    from conftest import ROOT
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


# ---- streams, graphs, and a run of them ----------------------------------------------------------------------------


@gpu
def test_calls_on_other_streams_and_in_graphs():
    tokens, experts, k, hidden = 600, 32, 8, 256
    logits = torch.randn(tokens, experts, generator=gen(1)).cuda()
    x = torch.randn(tokens, hidden, generator=gen(2)).to(torch.bfloat16).cuda()

    def step():
        ids, w = route_tokens(logits, k)
        rows, order = sort_tokens(x, ids, experts)
        return (ids, w, rows, *order, unsort_tokens(rows, order, w))

    def fresh(seed):
        logits.copy_(torch.randn(tokens, experts, generator=gen(seed)))
        x.copy_(torch.randn(tokens, hidden, generator=gen(seed + 1)))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graphs, outs = [], []
    for _ in range(2):                                                    # two captures, replayed at the same time
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (10, 20):
        fresh(seed)
        torch.cuda.synchronize()
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(want, out))


@gpu
def test_a_captured_training_step():
    tokens, experts, k, hidden = 64, 16, 4, 128
    logits = torch.randn(tokens, experts, generator=gen(1)).cuda().requires_grad_()
    x = torch.randn(tokens, hidden, generator=gen(2)).cuda().requires_grad_()
    dy = torch.randn(tokens, hidden, generator=gen(3)).cuda()

    def step():
        ids, w = route_tokens(logits, k)
        rows, order = sort_tokens(x, ids, experts, alignment=16)
        return torch.autograd.grad(unsort_tokens(rows * 2, order, w), [logits, x], dy)

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@gpu
def test_an_expert_layer_out_of_the_public_calls():
    """route -> sort -> up, SwiGLU, down -> back, against the layer class on the same weights: the same rows in the same order."""
    from nvfp4_cutlass_b200.ep import ExpertParallelMoE
    tokens, experts, k, hidden, inter = 300, 8, 2, 512, 256
    g = gen(5)
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16).cuda()
    up = nvfp4_gemm.quantize_weight_nvfp4((torch.randn(experts, 2 * inter, hidden, generator=g) * 0.05).to(torch.bfloat16).cuda())
    down = nvfp4_gemm.quantize_weight_nvfp4((torch.randn(experts, hidden, inter, generator=g) * 0.05).to(torch.bfloat16).cuda())
    ids, w = route_tokens(torch.randn(tokens, experts, generator=g).cuda(), k)
    rows, order = sort_tokens(x, ids, experts)
    h = torch.empty(rows.shape[0], 2 * inter, dtype=torch.bfloat16, device="cuda")
    nvfp4_gemm.m_grouped_bf16_dual_nvfp4_gemm_contiguous(rows, *up, h, order.m_indices)
    out = torch.empty(rows.shape[0], hidden, dtype=torch.bfloat16, device="cuda")
    _C.m_grouped_swiglu_dual_nvfp4_gemm_contiguous(h, *down, out, order.m_indices)
    y = unsort_tokens(out, order, w)
    layer = ExpertParallelMoE(experts, hidden, inter, up, down)
    assert torch.equal(y, layer(x, ids, w))


# ---- the calls in binding.cpp ----------------------------------------------------------------------------------------


def test_the_binding_takes_no_host_tensors_and_no_odd_arguments():
    _C.lib()
    b = _C._binding
    assert b is not None
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    assert b.route(x, 2, 0, 1) is None and b.route(None, 2, 0, 1) is None and b.route(x, "2", 0, 1) is None and b.route(x) is None
    assert b.sort(x, ids, 4, 16) is None and b.sort(x, None, 4, 16) is None and b.sort(x, ids, -4, 16) is None
    assert b.unsort(x, ids, ids, None) is None and b.unsort(x, ids, 3, None) is None and b.unsort(x) is None
    assert b.linear(x, x, None, None, 0, 0) is None and b.linear(x, x, None, None, 1 << 40, 0) is None and b.linear(x) is None
    with pytest.raises(TypeError):
        b.bind_operators(1)
    with pytest.raises(TypeError):
        b.bind_operators(*[0] * 10)


@gpu
def test_the_binding_gives_the_general_way_s_results(monkeypatch):
    g = gen(6)
    logits, x = torch.randn(50, 24, generator=g).cuda(), torch.randn(50, 72, generator=g).to(torch.bfloat16).cuda()
    w, bias = torch.randn(40, 72, generator=g).to(torch.bfloat16).cuda(), torch.randn(40, generator=g).to(torch.bfloat16).cuda()
    residual = torch.randn(50, 40, generator=g).cuda()

    def calls():
        ids, weights = route_tokens(logits, 3, scores="sigmoid", renormalize=False)
        rows, order = sort_tokens(x, ids, 24, alignment=16)
        return [ids, weights, rows, *order, unsort_tokens(rows, order, weights), unsort_tokens(rows, order),
                nvfp4_gemm.linear(x, w, bias, residual, activation="silu", out_dtype=torch.float32), nvfp4_gemm.linear(x, w)]

    _C.lib()
    assert _C._binding is not None
    fast = calls()
    # what it leaves to the general way: strided index tensors, empty ones
    b, ids = _C._binding, fast[0]
    assert b.sort(x, ids.t().contiguous().t(), 24, 16) is None and b.linear(x[:0], w, None, None, 0, 0) is None
    assert torch.equal(sort_tokens(x, ids.t().contiguous().t(), 24, alignment=16)[0], fast[2])
    with pytest.raises(RuntimeError, match="multiple of 8"):
        nvfp4_gemm.linear(x[:, :60], w[:, :60])
    monkeypatch.setattr(_C, "_binding", None)
    assert all(torch.equal(a, b) for a, b in zip(fast, calls()))


@gpu
def test_the_binding_s_gradients_are_the_general_way_s(monkeypatch):
    g = gen(7)
    leaf = lambda *shape, dtype=torch.bfloat16: torch.randn(*shape, generator=g).to(dtype).cuda().requires_grad_()
    logits, x, w, bias, residual = leaf(50, 24, dtype=torch.float32), leaf(50, 72), leaf(41, 72), leaf(41), leaf(50, 41, dtype=torch.float32)
    gw, gr, gy, gd = (torch.randn(*s, generator=g).cuda() for s in ((50, 3), (50, 72), (50, 72), (50, 41)))

    def grads():
        out = []
        ids, weights = route_tokens(logits, 3, scores="sigmoid")
        out += torch.autograd.grad(weights, logits, gw, retain_graph=True)
        rows, order = sort_tokens(x, ids, 24, alignment=16)
        y = unsort_tokens(rows, order, weights)
        out += torch.autograd.grad(y, [x, logits, rows], gy.bfloat16(), retain_graph=True)
        out += torch.autograd.grad(unsort_tokens(rows, order), rows, gy.bfloat16(), retain_graph=True)
        for act in ("none", "silu"):
            d = nvfp4_gemm.linear(x, w, bias, residual, activation=act, out_dtype=torch.float32)
            out += torch.autograd.grad(d, [x, w, bias, residual], gd, retain_graph=True)
            out += torch.autograd.grad(d, [residual], gd, retain_graph=True)
            out += torch.autograd.grad(nvfp4_gemm.linear(x.detach(), w, bias, activation=act), [w], gd.bfloat16())
        # a second derivative is an error, not nothing
        (first,) = torch.autograd.grad(weights.sum(), logits, create_graph=True)
        with pytest.raises(RuntimeError, match="once|does not require grad"):
            first.sum().backward()
        return out

    _C.lib()
    assert _C._binding is not None
    fast = grads()
    monkeypatch.setattr(_C, "_binding", None)
    slow = grads()
    assert len(fast) == len(slow) and all(torch.equal(a, b) for a, b in zip(fast, slow))


@gpu
def test_the_binding_records_calls_with_and_without_their_optional_arguments():
    _C.lib()
    b = _C._binding
    x = torch.randn(20, 64, generator=gen(1)).half().cuda().requires_grad_()
    w, bias, residual = x.detach()[:16].clone(), x.detach()[0, :16].clone(), torch.zeros(20, 16, dtype=torch.float16, device="cuda")
    for args in ((None, None), (bias, None), (None, residual), (bias, residual)):
        d = b.linear(x, w, *args, 4, 0)
        assert d is not None and torch.autograd.grad(d.sum(), x)[0].shape == x.shape
    rows, place, source, _ = b.sort(x, some_ids(20, 2, 4, 1, "uniform").cuda(), 4, 16)
    for weights in (None, torch.rand(20, 2, device="cuda")):
        y = b.unsort(rows, place, source, weights)
        assert y is not None and torch.autograd.grad(y.sum(), x, retain_graph=True)[0].shape == x.shape
    ids, weights = b.route(x, 4, 0, 1)
    assert torch.autograd.grad(weights.sum(), x)[0].shape == x.shape


@gpu
def test_what_is_not_differentiated_costs_nothing():
    x = torch.randn(6, 8, generator=gen(1)).cuda().requires_grad_()
    rows, order = sort_tokens(x, some_ids(6, 2, 4, 1, "uniform").cuda(), 4, alignment=16)
    assert rows.requires_grad and not any(t.requires_grad for t in order)
    ids, weights = route_tokens(x, 2)
    assert weights.requires_grad and not ids.requires_grad
    with torch.no_grad():
        assert not sort_tokens(x, ids, 8)[0].requires_grad and not route_tokens(x, 2)[1].requires_grad


# Orders that the caller has changed or made: what the forward sum takes from a row is what its gradient gets, whoever made the order
def hand_made(kind, ids, experts, alignment):
    place, source, m_indices = order_by_loops(ids, experts, alignment)
    h = len(ids) // 2
    if kind == "first half":
        place = place[:h]
    elif kind == "second half":
        place = place[h:]
    elif kind == "dropped late":
        place = place.masked_fill(torch.rand(place.shape, generator=gen(8)) < 0.4, -1)
    elif kind == "dropped all":
        place = torch.full_like(place, -1)
    elif kind == "one row for many":                                     # every third pair names one of three rows, some names are no rows
        place.view(-1)[::3] = torch.tensor([2, 5, len(source) - 1]).repeat(place.numel())[:place.view(-1)[::3].numel()]
        place.view(-1)[1::7] = len(source) + 3
    elif kind == "twice in a token":
        place[:, 1] = place[:, 0]
    elif kind == "shuffled":
        place = place[torch.randperm(len(place), generator=gen(9))]
    return TokenOrder(place, source, m_indices)


HAND_MADE = ["first half", "second half", "dropped late", "dropped all", "one row for many", "twice in a token", "shuffled"]


@gpu
@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("kind", HAND_MADE)
@pytest.mark.parametrize("tokens, k, experts, hidden", [(5, 2, 3, 8), (40, 4, 8, 70), (301, 6, 64, 520), (3000, 3, 16, 33)])
def test_gradients_of_orders_made_by_hand(tokens, k, experts, hidden, kind, binding, monkeypatch):
    _C.lib()
    if not binding:
        monkeypatch.setattr(_C, "_binding", None)
    order = hand_made(kind, some_ids(tokens, k, experts, 4, "uniform"), experts, 16)
    place, m = order.place, len(order.source)
    on_gpu = TokenOrder(*(t.cuda() for t in order))
    for dtype in ALL_TYPES:
        rows, w = torch.randn(m, hidden, generator=gen(1)).to(dtype), torch.randn(place.shape, generator=gen(2))
        dy = torch.randn(len(place), hidden, generator=gen(3)).to(dtype)
        for weights in (w, None):
            leaves = [rows.cuda().requires_grad_()] + ([weights.cuda().requires_grad_()] if weights is not None else [])
            y = unsort_tokens(leaves[0], on_gpu, *leaves[1:])
            live = (place >= 0) & (place < m)
            named = torch.where(live, place, -1)
            assert (y.detach().cpu().double() - sum_by_loops(rows, named, weights)).abs().le(sum_bound(rows, named, weights, dtype)).all()
            for again in range(2):
                stale = torch.full((m, hidden), float("nan"), dtype=dtype, device="cuda")      # what the next allocation of that size finds
                del stale
                grads = torch.autograd.grad(y, leaves, dy.cuda(), retain_graph=True)
                # drows[r]: the sum over the pairs that name r, in FP32, rounded once
                scale = (weights if weights is not None else torch.ones(place.shape)).double()
                terms = (scale[..., None] * dy.double()[:, None, :])[live]
                want = torch.zeros(m, hidden, dtype=torch.float64).index_add_(0, place[live], terms)
                size = torch.zeros(m, hidden, dtype=torch.float64).index_add_(0, place[live], terms.abs())
                count = torch.zeros(m, dtype=torch.float64).index_add_(0, place[live], torch.ones(int(live.sum()), dtype=torch.float64))
                tolerance = size * (count[:, None] * 2.0 ** -24 + 1.01 * HALF_STEP[dtype]) + (2.0 ** -25 if dtype == torch.float16 else 1e-40)
                assert (grads[0].cpu().double() - want).abs().le(tolerance).all()
                first = grads[0] if again == 0 else first
                assert torch.equal(grads[0], first)
                if weights is not None:
                    dots = torch.where(live[..., None], rows.double()[place.clamp(0, m - 1)], 0.0) * dy.double()[:, None, :]
                    assert (grads[1].cpu().double() - dots.sum(dim=2)).abs().le(dots.abs().sum(dim=2) * (hidden + 16) * 2.0 ** -24 + 1e-40).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("binding", [True, False])
def test_tangents_of_forward_mode_are_refused_not_lost(device, binding, monkeypatch):
    _C.lib()
    if not binding:
        monkeypatch.setattr(_C, "_binding", None)
    m = 16
    x, w = torch.randn(m, 8, device=device).to(torch.bfloat16), torch.rand(m, 2, device=device)
    order = TokenOrder(torch.zeros(m, 2, dtype=torch.int64, device=device), torch.zeros(m, dtype=torch.int32, device=device),
                       torch.zeros(m, dtype=torch.int32, device=device))
    bias, residual = torch.zeros(m, device=device, dtype=torch.bfloat16), torch.zeros(m, m, device=device, dtype=torch.bfloat16)
    calls = [(lambda t: route_tokens(t, 2), x), (lambda t: sort_tokens(t, order.place, 4, alignment=8), x), (lambda t: unsort_tokens(t, order), x),
             (lambda t: unsort_tokens(x, order, t), w), (lambda t: linear(t, x), x), (lambda t: linear(x, t), x), (lambda t: linear(x, x, t), bias),
             (lambda t: linear(x, x, None, t), residual)]
    for call, primal in calls:
        for recorded in (False, True):
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(primal.clone().requires_grad_(recorded), torch.ones_like(primal))
                with pytest.raises(RuntimeError, match="forward mode"):
                    call(dual)
            if device == "cuda":
                with forward_ad.dual_level():                             # a tensor without a tangent is an ordinary one
                    call(primal)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (primal,), (torch.ones_like(primal),))


@gpu
@pytest.mark.parametrize("binding", [True, False])
def test_saved_tensors_may_be_kept_on_the_host(binding, monkeypatch):
    """What the nodes keep goes through the hooks on saved tensors, and comes back with strides of its own."""
    _C.lib()
    if not binding:
        monkeypatch.setattr(_C, "_binding", None)
    wide = torch.randn(40, 88, generator=gen(1)).to(torch.bfloat16).cuda().requires_grad_()
    logits, w = torch.randn(40, 9, generator=gen(2)).cuda().requires_grad_(), torch.randn(24, 72, generator=gen(3)).to(torch.bfloat16).cuda().requires_grad_()

    def step():
        x = wide[:, 8:80]
        ids, weights = route_tokens(logits[:, 1:], 3)
        rows, order = sort_tokens(x, ids, 8, alignment=16)
        y = linear(unsort_tokens(rows, order, weights), w, activation="gelu") + linear(x, w, activation="none")
        return torch.autograd.grad(y.float().square().sum(), [wide, logits, w])

    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@gpu
@pytest.mark.parametrize("binding", [True, False])
def test_function_transforms_are_refused(binding, monkeypatch):
    _C.lib()
    if not binding:
        monkeypatch.setattr(_C, "_binding", None)
    x = torch.randn(3, 16, 8, generator=gen(1)).to(torch.bfloat16).cuda()
    ids = torch.zeros(16, 2, dtype=torch.int64, device="cuda")
    rows, order = sort_tokens(x[0], ids, 4, alignment=8)
    for call in (lambda t: route_tokens(t, 2)[1], lambda t: sort_tokens(t, ids, 4, alignment=8)[0], lambda t: linear(t, x[0]),
                 lambda t: unsort_tokens(t[:1].expand(len(rows), -1).contiguous(), order)):
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x)
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call(t).float().sum())(x[0])


@gpu
@pytest.mark.parametrize("k", [1, 2, 6])
@pytest.mark.parametrize("ahead", [0.0, 6.0, 12.0, 16.0, 18.0, 24.0, 30.0])
def test_routing_gradient_of_a_confident_token(ahead, k):
    """One logit far above the rest: the chosen expert's gradient is what the others leave of its score, and keeps its digits."""
    for experts in (8, 33, 128, 1000):
        for dtype in ALL_TYPES:
            logits = (torch.randn(6, experts, generator=gen(experts)) * 0.5).to(dtype).float()
            logits[torch.arange(6), torch.arange(6) % experts] = 3.0 + ahead
            logits[5, 7] = -math.inf
            logits = logits.to(dtype)
            for grad in (torch.ones(6, k), torch.rand(6, k, generator=gen(k)) + 0.5, torch.randn(6, k, generator=gen(k + 1))):
                leaf = logits.cuda().requires_grad_()
                ids, weights = route_tokens(leaf, k, renormalize=False)
                (got,) = torch.autograd.grad(weights, leaf, grad.cuda())
                p = torch.softmax(logits.double(), dim=1)
                chosen = torch.zeros(6, experts, dtype=torch.float64).scatter_(1, ids.cpu(), 1.0)
                g = torch.zeros(6, experts, dtype=torch.float64).scatter_(1, ids.cpu(), grad.double())
                left = (p * (1 - chosen)).sum(dim=1, keepdim=True)
                # g_j - sum g p over the chosen i = sum p_i (g_j - g_i) + g_j * (what the others have of p); its terms may cancel, each is
                # off by its scores' bound
                differences = (p * chosen)[:, None, :] * (g[:, :, None] - g[:, None, :])
                want = p * torch.where(chosen > 0, differences.sum(dim=2) + g * left, -(g * p).sum(dim=1, keepdim=True))
                size = p * torch.where(chosen > 0, differences.abs().sum(dim=2) + (g * left).abs(), (g * p).abs().sum(dim=1, keepdim=True))
                # three scores to a product, FP32 differences of g, sums of up to k + 1 terms, one rounding
                bound = 3 * weight_bound(logits.double(), k) + (k + 8) * 2.0 ** -24
                tolerance = size * bound + want.abs() * 1.01 * HALF_STEP[dtype] + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
                off = (got.cpu().double() - want).abs()
                assert off.le(tolerance).all(), float((off / tolerance).max())


def test_expired_waits_of_the_sum_need_a_bound():
    for budget in (0, -1, 2000000001):
        assert "budget" in error_of(_C.lib().nvfp4_debug_unsort_expired(16, 8, 0, 64, 16, 16, 4, 1, 8, 16, budget, None))


@gpu
@pytest.mark.parametrize("tokens, k, hidden", [(1000, 8, 4096), (5000, 2, 64), (3000, 32, 1024), (3000, 6, 520)])
def test_what_an_expired_wait_of_the_sum_leaves_is_nan(tokens, k, hidden):
    """Rows that are never fetched: the kernel ends after half a millisecond, with NaN in place of sums, and the next call is an ordinary one."""
    ids = some_ids(tokens, k, 64, 1, "holes").cuda()
    w = torch.rand(tokens, k, generator=gen(2)).cuda()
    for dtype in ALL_TYPES:
        rows, order = sort_tokens(torch.randn(tokens, hidden, generator=gen(1)).to(dtype).cuda(), ids, 64, alignment=16)
        want = unsort_tokens(rows, order, w)
        y = _C.debug_unsort_expired(rows, order.place, w, 1_000_000)
        assert torch.isnan(y).all()
        assert torch.equal(unsort_tokens(rows, order, w), want)


@gpu
@pytest.mark.parametrize("binding", [True, False])
def test_tensors_that_stand_for_their_negatives(binding, monkeypatch):
    _C.lib()
    if not binding:
        monkeypatch.setattr(_C, "_binding", None)
    x = torch.randn(40, 16, generator=gen(1)).cuda()
    negative = torch._neg_view(x)
    assert torch.equal(route_tokens(negative, 3)[0], route_tokens(-x, 3)[0])
    ids = torch.zeros(40, 2, dtype=torch.int64, device="cuda")
    rows, order = sort_tokens(negative, ids, 2, alignment=16)
    assert torch.equal(rows, sort_tokens(-x, ids, 2, alignment=16)[0])
    w = torch.rand(40, 2, generator=gen(2)).cuda()
    assert torch.equal(unsort_tokens(torch._neg_view(rows), order, w), unsort_tokens(-rows, order, w))
    assert torch.equal(unsort_tokens(rows, order, torch._neg_view(w)), unsort_tokens(rows, order, -w))
    h = x.half()
    b = torch.randn(40, generator=gen(3)).half().cuda()
    r = torch.randn(40, 40, generator=gen(3)).half().cuda()
    n = torch._neg_view
    assert torch.equal(linear(n(h), h, n(b), n(r)), linear(-h, h, -b, -r)) and torch.equal(linear(h, n(h)), linear(h, -h))
    leaf = h.clone().requires_grad_()
    y = linear(leaf, h)
    assert torch.equal(torch.autograd.grad(y, leaf, n(r), retain_graph=True)[0], torch.autograd.grad(y, leaf, -r)[0])
