"""Rotary positions on the GPU against the rotation in 64 bits.

Tolerance: with u the unit roundoff of the tensor's type, one rounding of the
result (u·|y|) after fp32 arithmetic of two products and a sum (three roundings
of terms that |a|+|b| bounds, the table's factor at most 1.2), plus the least
fp16 subnormal's half."""
import pytest
import torch

import npu_flash_attention as nfa
import rotary

DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def exact(x, cos, sin, pos, interleaved, inverse=False):
    """x [B, H, S, D] and pos [B, S] -> (rotated, bound of |a| + |b|) in fp64."""
    x = x.detach().double()
    r = 2 * cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    if inverse:
        s = -s
    y, size = x.clone(), x.abs()
    ai, bi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., ai], x[..., bi]
    y[..., ai], y[..., bi] = a * c - b * s, a * s + b * c
    size = size.clone()
    size[..., ai] = size[..., bi] = a.abs() + b.abs()
    return y, size


def close(got, ref, size):
    tol = U[got.dtype] * ref.abs() + 4 * 1.2 * 2.0 ** -24 * size + 2.0 ** -25
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} entries off, worst {((got.double() - ref).abs() - tol).max().item():.3g}"


def make(B, Hq, Hkv, S, D, dtype, seq_major=True, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def one(H):
        if seq_major:
            return torch.randn(B, S, H, D, generator=g, device=DEV).to(dtype).transpose(1, 2)
        return torch.randn(B, H, S, D, generator=g, device=DEV).to(dtype)
    return one(Hq), one(Hkv)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,Hq,Hkv,S,D,R,interleaved", [
    (1, 1, 1, 1, 64, 64, False), (8, 32, 8, 1, 128, 128, False), (2, 5, 1, 33, 128, 64, True), (2, 4, 4, 17, 80, 80, False),
    (1, 3, 1, 129, 256, 128, False), (1, 2, 2, 7, 128, 34, False), (1, 2, 2, 7, 64, 18, True), (3, 2, 1, 5, 6, 2, True),
    (2, 16, 2, 1500, 128, 128, False), (2, 16, 4, 1500, 128, 128, True), (1, 1, 1, 3, 65, 64, False)])
def test_forward_and_gradient(dtype, B, Hq, Hkv, S, D, R, interleaved):
    cos, sin = rotary.rotary_table(R, S + 50, scaling="yarn", factor=4.0, device=DEV)
    q, k = make(B, Hq, Hkv, S, D, dtype, seq_major=S % 2 == 1)
    dq, dk = make(B, Hq, Hkv, S, D, dtype, seq_major=S % 2 == 0, seed=1)
    off = torch.arange(B, device=DEV, dtype=torch.int32) * 7
    pos = off[:, None].long() + torch.arange(S, device=DEV)
    q.requires_grad_(True), k.requires_grad_(True)
    qo, ko = rotary.rotary_embedding(q, k, cos, sin, offsets=off, interleaved=interleaved)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    for got, x, inv in ((qo, q, False), (ko, k, False), (gq, dq, True), (gk, dk, True)):
        close(got, *exact(x, cos, sin, pos, interleaved, inv))
    nfa.check_device_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(interleaved):
    """The map is linear, so a central difference has no truncation error at
    any step; what remains is the fp32 rounding of outputs of size ~5."""
    cos, sin = rotary.rotary_table(32, 40, device=DEV)
    q, _ = make(1, 2, 1, 9, 48, torch.float32, seed=3)
    w, _ = make(1, 2, 1, 9, 48, torch.float32, seed=4)
    q = q.contiguous().requires_grad_(True)
    (g,) = torch.autograd.grad((rotary.rotary_embedding(q, None, cos, sin, interleaved=interleaved)[0] * w).sum(), q)
    gen = torch.Generator(device=DEV).manual_seed(9)
    for _ in range(8):
        i = tuple(int(torch.randint(0, n, (1,), generator=gen, device=DEV)) for n in q.shape)
        with torch.no_grad():
            e = torch.zeros_like(q)
            e[i] = 1.0
            up, _ = rotary.rotary_embedding(q + e, None, cos, sin, interleaved=interleaved)
            down, _ = rotary.rotary_embedding(q - e, None, cos, sin, interleaved=interleaved)
            diff = ((up.double() - down.double()) * w.double()).sum() / 2
        assert abs(diff.item() - g[i].item()) < 48 * 8 * 2.0 ** -24 * 5


@pytest.mark.gpu
def test_broadcast_and_strided_inputs():
    """An expanded input's gradient is summed over the broadcast; q with a
    stride on its innermost dim takes the element-wise form."""
    cos, sin = rotary.rotary_table(64, 64, device=DEV)
    base = torch.randn(1, 1, 16, 64, device=DEV, requires_grad=True)
    out, _ = rotary.rotary_embedding(base.expand(2, 3, 16, 64), None, cos, sin)
    w = torch.randn_like(out)
    (g,) = torch.autograd.grad(out, base, w)
    pos = torch.arange(16, device=DEV)[None].expand(2, -1)
    ref, _ = exact(w, cos, sin, pos, False, True)
    # Six fp32 terms of size up to ~5 are summed.
    assert (g.double() - ref.sum((0, 1), keepdim=True)).abs().max() < 6 * 6 * 5 * 2.0 ** -24
    wide = torch.randn(2, 3, 16, 128, device=DEV).to(torch.bfloat16)[..., ::2]
    out, _ = rotary.rotary_embedding(wide, None, cos, sin)
    close(out, *exact(wide, cos, sin, pos, False))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved,R", [(False, 128), (True, 64), (False, 34)])
def test_positions_in_place_and_one_tensor(interleaved, R):
    cos, sin = rotary.rotary_table(R, 500, device=DEV)
    q, k = make(3, 4, 2, 21, 128, torch.bfloat16)
    pos = torch.randint(0, 400, (3, 21), device=DEV)
    off = torch.tensor([0, 99, 3], device=DEV)
    at = pos + off[:, None]
    want = [exact(t, cos, sin, at, interleaved) for t in (q, k)]
    for p in (pos, pos.to(torch.int32)):
        qo, ko = rotary.rotary_embedding(q, k, cos, sin, p, off, interleaved=interleaved)
        close(qo, *want[0]), close(ko, *want[1])
    none, only = rotary.rotary_embedding(None, k, cos, sin, pos, off, interleaved=interleaved)
    assert none is None and torch.equal(only, ko)
    row = pos[0].contiguous()
    qo, _ = rotary.rotary_embedding(q, None, cos, sin, row, interleaved=interleaved)
    close(qo, *exact(q, cos, sin, row[None].expand(3, -1), interleaved))
    q2, k2 = q.clone(), k.clone()
    got = rotary.rotary_embedding(q2, k2, cos, sin, pos, off, interleaved=interleaved, out=(q2, k2))
    assert got[0] is q2
    close(q2, *want[0]), close(k2, *want[1])


@pytest.mark.gpu
def test_positions_outside_the_table_are_reported():
    cos, sin = rotary.rotary_table(32, 10, device=DEV)
    q, k = make(1, 2, 1, 4, 64, torch.bfloat16)
    nfa.check_device_status(DEV)
    for bad in (10, -1, 2 ** 40):
        pos = torch.tensor([0, bad, 9, 1], device=DEV)
        qo, _ = rotary.rotary_embedding(q, k, cos, sin, pos)
        with pytest.raises(RuntimeError, match="outside its table"):
            nfa.check_device_status(DEV)
        assert qo[:, :, 1, :32].isnan().all() and torch.equal(qo[:, :, 1, 32:], q[:, :, 1, 32:])
        keep = [0, 2, 3]
        close(qo[:, :, keep], *exact(q[:, :, keep], cos, sin, pos[None, keep], False))
    nfa.check_device_status(DEV)


@pytest.mark.gpu
def test_empty_and_refused():
    cos, sin = rotary.rotary_table(64, 10, device=DEV)
    q = torch.randn(2, 4, 0, 64, device=DEV)
    assert rotary.rotary_embedding(q, None, cos, sin)[0].shape == q.shape
    q = torch.randn(2, 4, 5, 64, device=DEV)
    for kw, err in ((dict(positions=torch.zeros(4, dtype=torch.int64, device=DEV)), ValueError),
                    (dict(positions=torch.zeros(5, device=DEV)), ValueError),
                    (dict(offsets=torch.zeros(3, dtype=torch.int32, device=DEV)), ValueError),
                    (dict(offsets=torch.zeros(2, dtype=torch.int32)), RuntimeError),
                    (dict(out=(q[:1], None)), ValueError)):
        with pytest.raises(err):
            rotary.rotary_embedding(q, None, cos, sin, **kw)
    with pytest.raises(AssertionError):
        rotary.rotary_embedding(q[..., :62], None, cos, sin)
    with pytest.raises(ValueError):
        rotary.rotary_embedding(q, None, cos.half(), sin.half())
    with pytest.raises(RuntimeError):
        rotary.rotary_embedding(q, q.half(), cos, sin)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        rotary.rotary_embedding(q.double(), None, cos, sin)
    with pytest.raises(ValueError, match="not differentiable"):
        rotary.rotary_embedding(q.requires_grad_(True), None, cos, sin, out=(torch.empty_like(q), None))


@pytest.mark.gpu
def test_other_streams():
    cos, sin = rotary.rotary_table(128, 300, device=DEV)
    q, k = make(4, 8, 2, 257, 128, torch.bfloat16)
    want = rotary.rotary_embedding(q, k, cos, sin)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = rotary.rotary_embedding(q, k, cos, sin)
    st.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_gradient_of_the_gradient():
    """The backward is the transposed rotation, differentiable in its turn: the
    gradient of <dq, v> in the output gradient is the rotation of v."""
    cos, sin = rotary.rotary_table(64, 40, device=DEV)
    q, k = make(2, 3, 1, 20, 64, torch.float32, seed=5)
    v, u = make(2, 3, 1, 20, 64, torch.float32, seed=6)
    q.requires_grad_(True), k.requires_grad_(True)
    out = rotary.rotary_embedding(q, k, cos, sin)
    g = [torch.randn_like(t).requires_grad_(True) for t in out]
    dq, dk = torch.autograd.grad(out, (q, k), g, create_graph=True)
    gg = torch.autograd.grad((dq * v).sum() + (dk * u).sum(), g)
    pos = torch.arange(20, device=DEV)[None].expand(2, -1)
    for got, x in zip(gg, (v, u)):
        close(got, *exact(x, cos, sin, pos, False))


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1])
def test_gradient_of_one_output(which):
    """Only one of q', k' is used: the other input's gradient is None."""
    cos, sin = rotary.rotary_table(64, 40, device=DEV)
    q, k = make(1, 2, 2, 9, 64, torch.bfloat16, seed=7)
    q.requires_grad_(True), k.requires_grad_(True)
    out = rotary.rotary_embedding(q, k, cos, sin, interleaved=True)
    w = torch.randn_like(out[which])
    grads = torch.autograd.grad(out[which], (q, k), w, allow_unused=True)
    pos = torch.arange(9, device=DEV)[None]
    close(grads[which], *exact(w, cos, sin, pos, True, True))
    assert grads[1 - which] is None


@pytest.mark.gpu
def test_out_is_written_in_place_for_autograd():
    """A tensor that autograd has saved and out= overwrites: the backward raises."""
    cos, sin = rotary.rotary_table(64, 40, device=DEV)
    q, k = make(1, 2, 2, 9, 64, torch.float32)
    w = torch.ones_like(q, requires_grad=True)
    before = q._version, k._version
    y = (w * q).sum()
    with torch.no_grad():
        rotary.rotary_embedding(q, k, cos, sin, out=(q, k))
    assert q._version > before[0] and k._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        x = torch.randn(1, 2, 9, 64, device=DEV)
    rotary.rotary_embedding(x, None, cos, sin, out=(x, None))


@pytest.mark.gpu
def test_out_that_requires_a_gradient_is_refused():
    cos, sin = rotary.rotary_table(64, 40, device=DEV)
    q, k = make(1, 2, 2, 9, 64, torch.float32)
    for out in ((torch.empty_like(q).requires_grad_(True), torch.empty_like(k)), (torch.empty_like(q), torch.empty_like(k).requires_grad_(True))):
        with pytest.raises(ValueError, match="not differentiable"):
            rotary.rotary_embedding(q, k, cos, sin, out=out)
        with torch.no_grad():
            rotary.rotary_embedding(q, k, cos, sin, out=out)


@pytest.mark.gpu
def test_a_backward_that_fails_raises():
    """The backward runs on autograd's own thread, without the interpreter's
    lock; an error there comes back as an exception (here from saved positions
    of another dtype)."""
    cos, sin = rotary.rotary_table(64, 40, device=DEV)
    q, _ = make(1, 2, 2, 9, 64, torch.float32)
    q.requires_grad_(True)
    pos = torch.arange(9, device=DEV)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.double() if t.dtype == torch.int64 else t):
        out, _ = rotary.rotary_embedding(q, None, cos, sin, pos)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="int32 or int64"):
        out.sum().backward()
    assert q.grad is None
    out, _ = rotary.rotary_embedding(q, None, cos, sin, pos)
    out.sum().backward()
    assert q.grad is not None


@pytest.mark.gpu
def test_out_may_not_overlap_but_in_place():
    cos, sin = rotary.rotary_table(64, 40, device=DEV)
    flat = torch.randn(4, 2, 2, 9, 64, device=DEV)
    q, k, a, b = flat
    late = flat.view(-1)[64:64 + q.numel()].view(q.shape)       # q, a row later
    wide = torch.empty(2, 1, 9, 64, device=DEV).expand(2, 2, 9, 64)
    turned = q.view(2, 9, 2, 64).transpose(1, 2)                # q's memory in another order
    for out in ((late, b), (wide, b), (turned, b), (k, q), (k, b), (a, q), (a, a), (a, flat.view(-1)[2 * q.numel() + 64:][:k.numel()].view(k.shape))):
        with pytest.raises(ValueError, match="overlap|share memory"):
            rotary.rotary_embedding(q, k, cos, sin, out=out)
    want = rotary.rotary_embedding(q, k, cos, sin)
    for out in ((a, b), (a, k.clone()), (q.clone(), b)):
        rotary.rotary_embedding(q, k, cos, sin, out=out)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    # In place: dense, one of the two, and interleaved in one projection's output.
    x, y = q.clone(), k.clone()
    rotary.rotary_embedding(x, y, cos, sin, out=(x, a))
    assert torch.equal(x, want[0]) and torch.equal(a, want[1])
    both = torch.cat((q, k), 1).transpose(1, 2).contiguous()    # [B, S, Hq + Hkv, D]
    x, y = both.transpose(1, 2).split(2, 1)
    rotary.rotary_embedding(x, y, cos, sin, out=(x, y))
    assert torch.equal(x, want[0]) and torch.equal(y, want[1])
    with pytest.raises(ValueError, match="overlap"):
        rotary.rotary_embedding(x, y, cos, sin, out=(y, x))
    # One head: its stride says nothing.
    x = q[:, :1].clone()
    other = x.as_strided(x.shape, (x.stride(0), 7, 64, 1))
    rotary.rotary_embedding(x, None, cos, sin, out=(other, None))
    assert torch.equal(x, want[0][:, :1])


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1])
def test_an_input_without_gradient_gets_none(which):
    """Its output requires none either, and the backward turns the other's alone."""
    cos, sin = rotary.rotary_table(64, 40, device=DEV)
    pair = list(make(1, 2, 1, 9, 64, torch.bfloat16, seed=8))
    pair[which].requires_grad_(True)
    out = rotary.rotary_embedding(*pair, cos, sin)
    assert out[which].requires_grad and not out[1 - which].requires_grad
    w = torch.randn_like(out[which])
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    (g,) = torch.autograd.grad((out[which],), (pair[which],), (w,))
    assert torch.cuda.memory_stats()["allocation.all.allocated"] - before == 1
    close(g, *exact(w, cos, sin, torch.arange(9, device=DEV)[None], False, True))
    # Through a sum of both outputs, and through a second derivative.
    out = rotary.rotary_embedding(*pair, cos, sin)
    (g,) = torch.autograd.grad(sum((t.float() ** 2).sum() for t in out), pair[which], create_graph=True)
    assert g.requires_grad and torch.autograd.grad(g.float().sum(), pair[which])[0] is not None


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_a_key_alone_costs_what_a_query_alone_does(interleaved):
    """The same tensor in either place takes the same (vector) form of the kernel."""
    cos, sin = rotary.rotary_table(128, 4096, device=DEV)
    x, _ = make(4, 32, 1, 4096, 128, torch.bfloat16)
    out = torch.empty_like(x)

    def best(call):
        times = []
        for _ in range(8):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record(), call(), b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)
    alone = best(lambda: rotary.rotary_embedding(x, None, cos, sin, interleaved=interleaved, out=(out, None)))
    want = out.clone()
    key = best(lambda: rotary.rotary_embedding(None, x, cos, sin, interleaved=interleaved, out=(None, out)))
    assert torch.equal(out, want)
    # The element-wise form takes several times as long; boxes vary by a few percent.
    assert key < 1.5 * alone, (key, alone)
