"""The head losses and the scaled embedding on the GPU against plain implementations in 64 bits.

Tolerances, fixed by the formats before any run. Norm-wise for gradients: bf16 rounds with a relative error of at
most 2^-9, once in G and once in the result, and the stored distances add 3.4e-4, so 2 * 2^-9 + 3.4e-4 < 4.5e-3.
Losses are fp32 from fp32 accumulators: 2e-5 of the largest magnitude entering them (logits and losses).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

GRAD_TOL = 4.5e-3
LOSS_TOL = 2e-5


def rel(a, b):
    a, b = a.double(), b.double()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def head_inputs(T, H, V, seed=0, scale=None, lean=6.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + T * 7919 + H * 31 + V)
    w = torch.randn(V, H, device="cuda", generator=g) * (scale or 0.05)
    labels = torch.randint(0, V, (T,), device="cuda", generator=g)
    h = torch.randn(T, H, device="cuda", generator=g)
    h = h + lean * torch.rand(T, 1, device="cuda", generator=g) * w[labels] / w[labels].norm(dim=1, keepdim=True)
    return h.bfloat16(), w.bfloat16(), labels


def ce64(h, w, labels, ignore=-100, upstream=None):
    """(row losses, dh, dw) in 64 bits for the given per-row upstream gradient (mean over live rows if None)."""
    live = labels != ignore
    h64, w64 = h.double(), w.double()
    hl = h64[live]
    logp = torch.log_softmax(hl @ w64.t(), 1)
    rows = torch.zeros(h.shape[0], dtype=torch.float64, device=h.device)
    rows[live] = -logp.gather(1, labels[live][:, None])[:, 0]
    up = torch.full_like(rows, 1.0 / max(1, int(live.sum()))) if upstream is None else upstream.double()
    G = logp.exp()
    G[torch.arange(G.shape[0], device=h.device), labels[live]] -= 1
    G = G * up[live][:, None]
    dh = torch.zeros_like(h64)
    dh[live] = G @ w64
    return rows, dh, G.t() @ hl


def kd64(h, w, values, indices, tau, upstream=None):
    V = w.shape[0]
    there = (indices >= 0) & (indices < V) & (values != -math.inf)
    live = there.any(1)
    h64, w64 = h.double(), w.double()
    logp = torch.log_softmax(h64[live] @ w64.t() / tau, 1)
    score = (values[live].double() / tau).masked_fill(~there[live], -math.inf)
    logq = torch.log_softmax(score, 1)
    q = logq.exp()
    pick = torch.where(there[live], indices[live].long(), 0)
    rows = torch.zeros(h.shape[0], dtype=torch.float64, device=h.device)
    terms = torch.where(there[live], q * (logq.masked_fill(~there[live], 0) - logp.gather(1, pick)), 0.0)
    rows[live] = tau * tau * terms.sum(1)
    up = torch.full_like(rows, 1.0 / max(1, int(live.sum()))) if upstream is None else upstream.double()
    G = logp.exp().scatter_add(1, pick, -q) * tau * up[live][:, None]
    dh = torch.zeros_like(h64)
    dh[live] = G @ w64
    return rows, dh, G.t() @ h64[live]


def check(status=True):
    from nano_train_b200.ops import check_status
    torch.cuda.synchronize()
    check_status(0)


def loss_close(got, want, h, w):
    top = float((h.double().abs().max() * 0 + want.abs().max()).item()) + 10.0
    assert got.dtype == torch.float32
    assert (got.double() - want).abs().max().item() <= LOSS_TOL * top, (got, want)


SIZES = [(1, 8, 1), (1, 64, 257), (2, 64, 2), (17, 264, 1000), (63, 128, 255), (64, 128, 256), (65, 256, 5003),
         (129, 1032, 511), (256, 512, 1024), (257, 768, 2051), (700, 64, 777), (600, 2304, 1025)]


@pytest.mark.parametrize("T,H,V", SIZES)
@pytest.mark.parametrize("masked", ["none", "some"])
def test_cross_entropy_mean(T, H, V, masked):
    from nano_train_b200 import ops
    h, w, lab = head_inputs(T, H, V)
    if masked == "some":
        lab = torch.where(torch.arange(T, device="cuda") % 3 == 1, -100, lab)
    h.requires_grad_(True)
    w.requires_grad_(True)
    loss = ops.linear_cross_entropy(h, w, lab)
    (loss * 1.0).backward()
    rows, dh, dw = ce64(h.detach(), w.detach(), lab)
    check()
    live = max(1, int((lab != -100).sum()))
    loss_close(loss.detach(), rows.sum() / live, h.detach(), w.detach())
    if V > 1:
        assert rel(h.grad, dh) < GRAD_TOL
        assert rel(w.grad, dw) < GRAD_TOL
    else:  # one word: the loss is 0 whatever the inputs
        assert h.grad.abs().max() < 1e-6 and w.grad.abs().max() < 1e-6
    assert (h.grad[lab == -100] == 0).all()


@pytest.mark.parametrize("T,H,V", [(1, 64, 257), (65, 256, 5003), (257, 768, 2051), (600, 1024, 1025)])
def test_cross_entropy_rows_and_scores(T, H, V):
    from nano_train_b200 import ops
    h, w, lab = head_inputs(T, H, V, seed=1)
    lab = torch.where(torch.arange(T, device="cuda") % 5 == 2, -100, lab)
    up = torch.randn(T, device="cuda")
    with torch.no_grad():
        scored = ops.linear_cross_entropy(h, w, lab, reduction="none")
    h.requires_grad_(True)
    w.requires_grad_(True)
    rows = ops.linear_cross_entropy(h, w, lab, reduction="none")
    rows.backward(up)
    want, dh, dw = ce64(h.detach(), w.detach(), lab, upstream=up)
    check()
    assert torch.equal(scored, rows.detach())
    loss_close(rows.detach(), want, h.detach(), w.detach())
    assert rel(h.grad, dh) < GRAD_TOL and rel(w.grad, dw) < GRAD_TOL


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_chunks_main_grad_and_upstream(reduction):
    """Several chunks of tokens (a 1 MB workspace holds 256 of them), an upstream gradient and a main_grad."""
    from nano_train_b200 import ops
    T, H, V = 900, 192, 3001
    h, w, lab = head_inputs(T, H, V, seed=2)
    lab[300:620] = -100  # live tokens end inside the third chunk; the fourth has none
    live = int((lab != -100).sum())
    want, dh, dw = ce64(h, w, lab, upstream=torch.full((T,), 0.75 / (live if reduction == "mean" else 1),
                                                       device="cuda", dtype=torch.float64))
    for main in (False, True):
        hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        calls = []
        if main:
            ww.main_grad = torch.full((V, H), 0.5, device="cuda")
            ww._ntb_grad_ready_hook = calls.append
        loss = ops.linear_cross_entropy(hh, ww, lab, reduction=reduction, max_workspace_mb=1)
        (loss * 0.75).backward()
        check()
        loss_close(loss.detach(), want.sum() / (live if reduction == "mean" else 1), h, w)
        assert rel(hh.grad, dh) < GRAD_TOL
        if main:
            assert ww.grad is None and len(calls) == 1 and calls[0] is ww
            # fp32 results on top of 0.5: only G's rounding and the addition's
            assert (ww.main_grad.double() - 0.5 - dw).norm() / dw.norm() < GRAD_TOL
        else:
            assert rel(ww.grad, dw) < GRAD_TOL


def test_all_tokens_masked_and_none_given():
    from nano_train_b200 import ops
    for T in (0, 1, 70, 300):
        h, w, _ = head_inputs(max(T, 1), 64, 500)
        h, w = h[:T].clone().requires_grad_(True), w.requires_grad_(True)
        lab = torch.full((T,), -100, device="cuda")
        loss = ops.linear_cross_entropy(h, w, lab)
        loss.backward()
        check()
        assert loss.item() == 0.0
        assert h.grad.shape == h.shape and (h.grad == 0).all() and (w.grad == 0).all()
        idx = torch.full((T, 3), -1, device="cuda")
        w.grad = None
        loss = ops.linear_distillation(h, w, torch.zeros(T, 3, device="cuda"), idx)
        loss.backward()
        check()
        assert loss.item() == 0.0 and (w.grad == 0).all()


def test_masked_tokens_may_hold_nan():
    from nano_train_b200 import ops
    h, w, lab = head_inputs(130, 128, 999, seed=3)
    lab[::4] = -100
    clean = h.clone()
    h[::4] = float("nan")
    h[4] = float("inf")
    clean[::4] = 0
    for reduction in ("mean", "none"):
        a, wa = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        b, wb = clean.clone().requires_grad_(True), w.clone().requires_grad_(True)
        la = ops.linear_cross_entropy(a, wa, lab, reduction=reduction)
        lb = ops.linear_cross_entropy(b, wb, lab, reduction=reduction)
        la.sum().backward()
        lb.sum().backward()
        check()
        assert torch.equal(la, lb) and torch.equal(a.grad, b.grad) and torch.equal(wa.grad, wb.grad)
        assert torch.isfinite(a.grad).all() and torch.isfinite(wa.grad).all()


@pytest.mark.parametrize("gain", [30.0, 400.0])
def test_large_logits(gain):
    """Logits of several hundred: probabilities of 0 and 1 exactly, targets far below the maximum."""
    from nano_train_b200 import ops
    T, H, V = 96, 256, 1500
    h, w, lab = head_inputs(T, H, V, seed=4)
    h = (h.float() * gain).bfloat16().requires_grad_(True)
    w.requires_grad_(True)
    loss = ops.linear_cross_entropy(h, w, lab)
    loss.backward()
    rows, dh, dw = ce64(h.detach(), w.detach(), lab)
    check()
    top = (h.detach().double() @ w.detach().double().t()).abs().max().item()
    assert abs(loss.item() - rows.mean().item()) <= LOSS_TOL * top
    # a logit's fp32 error of about 2^-23 * top turns into that relative error of a probability
    assert rel(h.grad, dh) < GRAD_TOL + 2 ** -20 * top and rel(w.grad, dw) < GRAD_TOL + 2 ** -20 * top


def test_minus_infinite_logits():
    """Rows of the head at -inf (a masked part of the vocabulary) have probability 0 and no NaN."""
    from nano_train_b200 import ops
    T, H, V = 40, 64, 1024
    h, w, lab = head_inputs(T, H, V, seed=5)
    h = h.abs()  # positive states, so that the product with -inf is -inf
    lab = lab % 256
    w[256:] = -float("inf")
    with torch.no_grad():
        rows = ops.linear_cross_entropy(h, w, lab, reduction="none")
    check()
    want, _, _ = ce64(h, w[:256], lab)
    loss_close(rows, want, h, w[:256])


def test_strides_streams_and_determinism():
    from nano_train_b200 import ops
    T, H, V = 200, 136, 1111
    h, w, lab = head_inputs(T, H, V, seed=6)
    base = ops.linear_cross_entropy(h, w, lab, reduction="none")
    wide = torch.zeros(T, 3 * H, device="cuda", dtype=torch.bfloat16)
    wide[:, H:2 * H] = h
    odd = torch.zeros(T, 2 * H + 3, device="cuda", dtype=torch.bfloat16)
    odd[:, 1:1 + H] = h
    for view in (wide[:, H:2 * H], odd[:, 1:1 + H], h.t().contiguous().t(), h.view(10, 20, H)):
        l = lab.view(view.shape[:-1])
        got = ops.linear_cross_entropy(view, w, l, reduction="none")
        assert got.shape == l.shape and torch.equal(got.view(-1), base)
    assert torch.equal(ops.linear_cross_entropy(h, w.t().contiguous().t(), lab, reduction="none"), base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for stream in (side, torch.cuda.current_stream()):
        with torch.cuda.stream(stream):
            hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
            loss = ops.linear_cross_entropy(hh, ww, lab)
            loss.backward()
            outs.append((loss.detach(), hh.grad, ww.grad))
    check()
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_one_sided_gradients_and_second_backward():
    from nano_train_b200 import ops
    T, H, V = 150, 256, 900
    h, w, lab = head_inputs(T, H, V, seed=7)
    _, dh, dw = ce64(h, w, lab)
    a = h.clone().requires_grad_(True)
    ops.linear_cross_entropy(a, w, lab).backward()
    assert rel(a.grad, dh) < GRAD_TOL
    b = w.clone().requires_grad_(True)
    ops.linear_cross_entropy(h, b, lab).backward()
    assert rel(b.grad, dw) < GRAD_TOL
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = ops.linear_cross_entropy(a, b, lab)
    first = torch.autograd.grad(loss, (a, b), torch.tensor(3.0, device="cuda"), retain_graph=True)
    second = torch.autograd.grad(loss, (a, b), torch.tensor(-2.0, device="cuda"))
    check()
    for x, y, want in zip(first, second, (dh, dw)):
        # 3 is no power of two: the ready gradients are rounded a second time
        assert rel(x, 3 * want) < GRAD_TOL + 2 ** -9 and rel(y, -2 * want) < GRAD_TOL


@pytest.mark.parametrize("kind", ["ce", "kd"])
def test_gradient_against_differences(kind):
    """Central differences of the fp32 loss along a direction; states and steps are multiples of 2^-4, exact in bf16."""
    from nano_train_b200 import ops
    T, H, V = 33, 128, 700
    h, w, lab = head_inputs(T, H, V, seed=8, lean=2.0)
    h = ((h.float() * 16).round().clamp(-64, 64) / 16).bfloat16()
    values = torch.randn(T, 5, device="cuda")
    idx = torch.stack([torch.randperm(V, device="cuda")[:5] for _ in range(T)])

    def f(x):
        if kind == "ce":
            return ops.linear_cross_entropy(x, w, lab, reduction="sum")
        return ops.linear_distillation(x, w, values, idx, temperature=1.5, reduction="sum")

    a = h.clone().requires_grad_(True)
    f(a).backward()
    d = a.grad.float().sign()  # the direction of steepest ascent among +-1
    eps = 2.0 ** -4
    up, down = (h.float() + eps * d).bfloat16(), (h.float() - eps * d).bfloat16()
    assert torch.equal(up.float() - h.float(), eps * d) and torch.equal(h.float() - down.float(), eps * d)
    with torch.no_grad():
        diff = (f(up).double() - f(down).double()) / (2 * eps)
    check()
    along = (a.grad.double() * d.double()).sum()
    # third-order term: a logit moves by at most eps sum |w| = 0.04 * 0.05 * 128 * 0.8 = 0.33 -> under 0.33^2 / 6 = 2 %
    assert abs(diff.item() / along.item() - 1) < 0.02


# ------------------------------------------------------------------------------------------------ distillation
@pytest.mark.parametrize("T,H,V,K,tau", [(1, 64, 300, 1, 1.0), (5, 128, 64, 64, 2.0), (70, 264, 1000, 7, 0.7),
                                         (129, 512, 5003, 33, 1.0), (300, 256, 2048, 200, 3.0), (40, 64, 4096, 1024, 1.0)])
def test_distillation(T, H, V, K, tau):
    from nano_train_b200 import ops
    h, w, _ = head_inputs(T, H, V, seed=9)
    g = torch.Generator(device="cuda").manual_seed(K)
    idx = torch.rand(T, V, device="cuda", generator=g).topk(K, dim=1).indices
    values = (torch.randn(T, K, device="cuda", generator=g) * 3).sort(1, descending=True).values
    idx[3::7] = -1                       # tokens without entries
    if K > 2:
        idx[1::5, K // 2:] = -1          # short lists
        idx[2::6, 0] = V + 3             # outside the vocabulary
        values[0::9, 1] = -math.inf
    for vd, idt in ((torch.float32, torch.int64), (torch.bfloat16, torch.int32), (torch.float16, torch.int64)):
        v = values.to(vd)
        hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = ops.linear_distillation(hh, ww, v, idx.to(idt), temperature=tau)
        loss.backward()
        rows, dh, dw = kd64(h, w, v, idx, tau)
        check()
        live = max(1, int(((idx >= 0) & (idx < V)).any(1).sum()))
        loss_close(loss.detach() / tau ** 2, rows.sum() / live / tau ** 2, h, w)
        assert rel(hh.grad, dh) < GRAD_TOL and rel(ww.grad, dw) < GRAD_TOL


def test_distillation_rows_duplicates_and_order():
    from nano_train_b200 import ops
    T, H, V, K = 64, 128, 1500, 12
    h, w, _ = head_inputs(T, H, V, seed=10)
    g = torch.Generator(device="cuda").manual_seed(0)
    idx = torch.randint(0, 40, (T, K), device="cuda", generator=g) * 37  # duplicates in most rows
    values = torch.randn(T, K, device="cuda", generator=g)
    up = torch.randn(T, device="cuda", generator=g)
    rows64, dh, dw = kd64(h, w, values, idx, 2.0, upstream=up)
    results = []
    for order in (torch.arange(K), torch.randperm(K, generator=torch.Generator().manual_seed(1))):
        hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        rows = ops.linear_distillation(hh, ww, values[:, order], idx[:, order], temperature=2.0, reduction="none")
        rows.backward(up)
        check()
        loss_close(rows.detach(), rows64, h, w)
        assert rel(hh.grad, dh) < GRAD_TOL and rel(ww.grad, dw) < GRAD_TOL
        results.append(rows.detach())
    # strided teacher tensors
    big = torch.zeros(T, 2 * K, device="cuda")
    big[:, ::2] = values
    assert torch.equal(ops.linear_distillation(h, w, big[:, ::2], idx, temperature=2.0, reduction="none"), results[0])


def test_distillation_of_itself_has_no_gradient():
    """A teacher whose K = V logits are the student's own: q = p, loss and gradient vanish up to rounding."""
    from nano_train_b200 import ops
    T, H, V = 50, 64, 512
    h, w, _ = head_inputs(T, H, V, seed=11)
    own = h.float() @ w.float().t()
    h.requires_grad_(True)
    loss = ops.linear_distillation(h, w, own, torch.arange(V, device="cuda").expand(T, V))
    loss.backward()
    check()
    assert abs(loss.item()) < 1e-5
    # p and q agree to fp32 rounding of logits of size 10: 1e-5 of each probability, summed against |w|
    assert h.grad.abs().max().item() < 1e-5 * w.float().abs().max().item()


# ------------------------------------------------------------------------------------------------ embedding
def embed64(ids, w, scale, start, dout):
    V = w.shape[0]
    table = torch.cat([w.double(), torch.zeros(1, w.shape[1], dtype=torch.float64, device=w.device)])
    row = ids.reshape(-1) - start
    row = torch.where((row < 0) | (row >= V), V, row)
    grad = torch.zeros_like(table)
    grad.index_put_((row,), dout.reshape(-1, w.shape[1]).double() * scale, accumulate=True)
    return (table[row] * scale).view(*ids.shape, -1), grad[:V]


@pytest.mark.parametrize("n,H,V", [(1, 1, 1), (1, 8, 1), (2, 64, 3), (31, 33, 7), (32, 256, 1), (33, 1032, 511),
                                   (65, 7, 512), (1000, 264, 513), (2049, 100, 130000), (5000, 1536, 300),
                                   (20000, 72, 262145)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("start", [0, 3])
def test_scaled_embedding(n, H, V, dtype, start):
    from nano_train_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(n + H + V)
    w = torch.randn(V, H, device="cuda", generator=g).to(dtype).requires_grad_(True)
    u = torch.rand(n, device="cuda", generator=g)
    ids = (torch.exp(u * math.log(V + 6.0)).long() - 1 + (start if V < 10 else 0))  # heavy-tailed, some outside
    dout = torch.randn(n, H, device="cuda", generator=g).to(dtype)
    for scale in (1.0, 2.5):
        w.grad = None
        out = ops.scaled_embedding(ids, w, scale, vocab_start=start)
        out.backward(dout)
        want, dw = embed64(ids, w.detach(), scale, start, dout)
        check()
        unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
        assert out.dtype == dtype and (out.double() - want).abs().max() <= unit * want.abs().max().clamp_min(1e-30)
        # fp32 sums of up to n terms, then one rounding to the type
        assert rel(w.grad, dw) < unit + 2.0 ** -24 * math.sqrt(n) + 1e-7
        untouched = torch.ones(V, dtype=torch.bool, device="cuda")
        local = ids - start
        untouched[local[(local >= 0) & (local < V)]] = False
        assert (w.grad[untouched] == 0).all()


def test_scaled_embedding_runs_main_grad_and_determinism():
    """One id in nearly every token: its run crosses hundreds of pieces."""
    from nano_train_b200 import ops
    n, H, V = 10000, 520, 1000
    g = torch.Generator(device="cuda").manual_seed(5)
    ids = torch.where(torch.rand(n, device="cuda", generator=g) < 0.9, 17, torch.randint(0, V, (n,), device="cuda"))
    for dtype in (torch.bfloat16, torch.float32):
        w = torch.randn(V, H, device="cuda", generator=g).to(dtype).requires_grad_(True)
        dout = torch.randn(n, H, device="cuda", generator=g).to(dtype)
        grads = []
        for _ in range(2):
            (dw,) = torch.autograd.grad(ops.scaled_embedding(ids, w, 0.25), (w,), dout)
            grads.append(dw)
        _, want = embed64(ids, w.detach(), 0.25, 0, dout)
        assert torch.equal(*grads)
        assert rel(grads[0], want) < (2.0 ** -8 if dtype == torch.bfloat16 else 1e-5)
        seen = []
        w.main_grad = torch.full((V, H), 2.0, device="cuda")
        w._ntb_grad_ready_hook = seen.append
        ops.scaled_embedding(ids.view(100, 100), w, 0.25).backward(dout.view(100, 100, H))
        check()
        assert w.grad is None and seen == [w]
        assert rel(w.main_grad - 2.0, want) < 1e-5


def test_scaled_embedding_broadcast_gradient_empty_and_other_ids():
    from nano_train_b200 import ops
    w = torch.randn(64, 48, device="cuda").bfloat16().requires_grad_(True)
    ids = torch.randint(0, 64, (3, 5), device="cuda")
    ops.scaled_embedding(ids, w, 3.0).sum().backward()  # a broadcast upstream gradient
    counts = torch.bincount(ids.view(-1), minlength=64).double()
    check()
    assert torch.equal(w.grad.double(), (counts * 3)[:, None].expand(64, 48))
    w.grad = None
    out = ops.scaled_embedding(torch.empty(0, dtype=torch.int64, device="cuda"), w, 3.0)
    out.sum().backward()
    assert out.shape == (0, 48) and (w.grad == 0).all()
    w.grad = None
    ops.scaled_embedding(torch.tensor([-1, 64, 2 ** 40, -2 ** 40], device="cuda"), w).sum().backward()
    check()
    assert (w.grad == 0).all()
    # the same rows as the unscaled lookup
    assert torch.equal(ops.scaled_embedding(ids, w), ops.embedding(ids, w))


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals_on_cuda():
    from nano_train_b200 import ops
    h, w, lab = head_inputs(8, 64, 100)
    with pytest.raises(TypeError):
        ops.linear_cross_entropy(h.float(), w.float(), lab)
    with pytest.raises(TypeError):
        ops.linear_cross_entropy(h, w.float(), lab)
    with pytest.raises(TypeError):
        ops.linear_cross_entropy(h, w, lab.int())
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(h[:, :60], w[:, :60], lab)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(h, w[:1].expand(2 ** 19 + 1, 64), lab)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(h, w, lab[:7])
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(h, w, lab.cpu())
    with pytest.raises(ValueError):
        ops.linear_distillation(h, w, torch.zeros(8, 1025, device="cuda"), torch.zeros(8, 1025, device="cuda").long())
    with pytest.raises(TypeError):
        ops.linear_distillation(h, w, torch.zeros(8, 2, device="cuda").double(),
                                torch.zeros(8, 2, device="cuda").long())
    with pytest.raises(TypeError):
        ops.scaled_embedding(lab, w.half())
    with pytest.raises(RuntimeError):  # no second derivative
        x = h.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(ops.linear_cross_entropy(x, w, lab), (x,), create_graph=True)
        g.sum().backward()
    check()
