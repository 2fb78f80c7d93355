"""First calls from threads that have not used the device yet: autograd's in a backward pass, threads of the caller's."""
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

SETUP = """
import threading
import torch, nvfp4_gemm
x = torch.randn(384, 512, device="cuda").to(torch.bfloat16)
w = torch.randn(256, 512, device="cuda").to(torch.bfloat16)
weights = nvfp4_gemm.quantize_weight_nvfp4(w[None].contiguous())
m_indices = nvfp4_gemm.make_m_indices([384]).cuda()
d = torch.empty(384, 256, device="cuda", dtype=torch.bfloat16)
ids = torch.zeros(384, 4, dtype=torch.int64, device="cuda")
logits = torch.randn(384, 16, device="cuda")
def gemm(**kw):
    nvfp4_gemm.m_grouped_bf16_dual_nvfp4_gemm_contiguous(x, *weights, d, m_indices, **kw)
    return d
def moved():
    rows, order = nvfp4_gemm.sort_tokens(x, ids, 4)
    return nvfp4_gemm.unsort_tokens(rows, order)
torch.cuda.synchronize()
def backward():                  # without an activation or a bias the first kernel is a product
    leaf = x.clone().requires_grad_()
    y = nvfp4_gemm.linear(leaf, w)
    return torch.autograd.grad(y, leaf, torch.ones_like(y))[0]
def in_a_thread(call):
    out = []
    t = threading.Thread(target=lambda: (out.append(call()), torch.cuda.synchronize()))
    t.start(); t.join()
    assert out, "the thread's call failed"
    return out[0].clone()
"""
BACKWARD = """
got = backward()
want = torch.ones(384, 256, device="cuda").bfloat16() @ w
assert (got.float() - want.float()).abs().max() <= 2 * 2.0 ** -8 * want.float().abs().max()      # two roundings of one sum
"""
CALLS = """
for call in (lambda: nvfp4_gemm.linear(x, w), gemm, lambda: gemm(tune_split_transform=2), lambda: gemm(tune_split_transform=2, tune_cluster=1),
             lambda: gemm(tune_swap_ab=1, m_alignment=128), moved, lambda: nvfp4_gemm.route_tokens(logits, 3)[1]):
    assert torch.equal(in_a_thread(call), call())
"""


@pytest.mark.parametrize("calls", [BACKWARD, CALLS], ids=["backward", "calls"])
def test_the_first_call_of_a_thread(calls):
    r = subprocess.run([sys.executable, "-c", SETUP + calls], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


def test_training_steps_of_several_threads_at_once():
    """Every thread trains on a stream of its own, sizes that differ, workspaces out of one pool: the bits of the steps one after the other."""
    import threading

    import torch

    from nvfp4_gemm import linear, route_tokens, sort_tokens, unsort_tokens

    def case(i):
        g = torch.Generator().manual_seed(i)
        dtype = (torch.bfloat16, torch.float16)[i % 2]
        tokens = 700 + 333 * i
        leaf = lambda *s, scale: (torch.randn(*s, generator=g) * scale).to(dtype).cuda().requires_grad_()
        leaves = [leaf(tokens, 256, scale=1.0), leaf(16, 256, scale=0.1), leaf(264, 256, scale=0.06), leaf(264, scale=0.1), leaf(256, 264, scale=0.06)]
        dy = (torch.randn(tokens, 256, generator=g) * (1.0, 1e-6)[i % 2]).cuda()
        return leaves, dy

    def step(leaves, dy):
        x, gate, w1, bias, w2 = leaves
        ids, weights = route_tokens(linear(x, gate, out_dtype=torch.float32), 4, renormalize=False)
        rows, order = sort_tokens(x, ids, 16, alignment=16)
        d = linear(linear(rows, w1, bias, activation="silu"), w2)
        y = linear(x, w2.detach()[:, :256].contiguous(), out_dtype=torch.float32) + unsort_tokens(d, order._replace(place=order.place.flip(1)), weights).float()
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    cases = [case(i) for i in range(4)]
    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    same = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(15):
                got = step(*cases[i])
                stream.synchronize()
                same.append(all(torch.equal(a, b) for a, b in zip(got, want[i])))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(same) == 4 * 15 and all(same)
