"""Refusals of the vocabulary operators that need no GPU, and the reference
that the GPU tests compare with, checked against itself."""
import ctypes

import numpy as np
import pytest
import torch

import vocabulary_reference as ref

F32, F64, I32, I64, F16, BF16 = 0, 1, 2, 3, 4, 5
E_INVALID, E_WORKSPACE, E_UNSUPPORTED = 1, 2, 3
# Addresses that no call below gets as far as using.
A, B, C = 1 << 20, 1 << 24, 1 << 28


def lookup(lib, dtype=F32, table=A, rows=8, width=4, stride=4, tdtype=I32,
           tokens=B, count=2, out=C):
    return lib.mgpu_b200_embedding_lookup(dtype, table, rows, width, stride,
                                          tdtype, tokens, count, 1.0, out, None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=F64), E_UNSUPPORTED), (dict(dtype=9), E_UNSUPPORTED),
    (dict(tdtype=F32), E_UNSUPPORTED), (dict(table=None), E_INVALID),
    (dict(tokens=None), E_INVALID), (dict(out=None), E_INVALID),
    (dict(stride=3), E_INVALID), (dict(count=-1), E_INVALID),
    (dict(rows=-1), E_INVALID), (dict(width=-1), E_INVALID),
    (dict(width=(1 << 20) + 1, stride=1 << 21), E_INVALID),
    (dict(table=A + 2), E_INVALID), (dict(out=C + 1), E_INVALID),
    (dict(tokens=B + 2), E_INVALID), (dict(tdtype=I64, tokens=B + 4), E_INVALID),
    (dict(out=A + 16), E_INVALID), (dict(rows=2**31 - 1), E_INVALID),
    (dict(count=0, tokens=None, out=None), 0), (dict(width=0, out=None), 0)])
def test_lookup_refusals(mgpu, change, code):
    assert lookup(mgpu.load_library(), **change) == code


def gradient(lib, dtype=BF16, grad=A, stride=4, width=4, tdtype=I64, tokens=B,
             count=2, rows=8, accumulate=0, odtype=BF16, out=C, ws=1 << 29,
             nbytes=1 << 30):
    return lib.mgpu_b200_embedding_gradient(
        dtype, grad, stride, width, tdtype, tokens, count, rows, 1.0,
        accumulate, odtype, out, ws, nbytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=F64), E_UNSUPPORTED), (dict(odtype=F16), E_UNSUPPORTED),
    (dict(dtype=F32, odtype=BF16), E_UNSUPPORTED),
    (dict(tdtype=F32), E_UNSUPPORTED), (dict(grad=None), E_INVALID),
    (dict(tokens=None), E_INVALID), (dict(out=None), E_INVALID),
    (dict(ws=None), E_INVALID), (dict(ws=(1 << 29) + 64), E_INVALID),
    (dict(nbytes=64), E_WORKSPACE), (dict(stride=2), E_INVALID),
    (dict(out=A), E_INVALID), (dict(count=-1), E_INVALID),
    (dict(count=2**31 - 1), E_INVALID), (dict(rows=0), 0),
    (dict(width=0), 0), (dict(accumulate=1, count=0), 0)])
def test_gradient_refusals(mgpu, change, code):
    assert gradient(mgpu.load_library(), **change) == code


def test_gradient_workspace_sizes(mgpu):
    size = mgpu.load_library().mgpu_b200_embedding_gradient_workspace_bytes
    assert 0 < size(0, 1, 1, 0) <= size(1000, 1000, 64, 0) < size(
        10000, 100000, 4096, 0) < 1 << 30
    assert size(-1, 8, 8, 0) == size(8, -1, 8, 0) == size(8, 8, -1, 0) == 0
    assert size(2**31 - 1, 2**31 - 1, 8, 0) == 0
    assert size(8, 8, (1 << 20) + 1, 0) == 0


def distill(lib, grad_too, dtype=F32, logits=A, stride=100, count=2, vocab=100,
            tdtype=I32, tokens=B, hdtype=F32, teacher=B + 4096, entries=4,
            temperature=1.0, weights=None, losses=C, grad=1 << 30,
            grad_stride=100):
    if not grad_too:
        return lib.mgpu_b200_distill_loss(
            dtype, logits, stride, count, vocab, tdtype, tokens, hdtype,
            teacher, entries, temperature, losses, None)
    return lib.mgpu_b200_distill_loss_gradient(
        dtype, logits, stride, count, vocab, tdtype, tokens, hdtype, teacher,
        entries, temperature, weights, losses, grad, grad_stride, None)


@pytest.mark.parametrize("grad_too", [False, True])
@pytest.mark.parametrize("change,code", [
    (dict(dtype=F64), E_UNSUPPORTED), (dict(hdtype=I32), E_UNSUPPORTED),
    (dict(tdtype=F16), E_UNSUPPORTED), (dict(logits=None), E_INVALID),
    (dict(tokens=None), E_INVALID), (dict(teacher=None), E_INVALID),
    (dict(losses=None), E_INVALID), (dict(stride=99), E_INVALID),
    (dict(count=-1), E_INVALID), (dict(vocab=-1), E_INVALID),
    (dict(entries=-1), E_INVALID), (dict(entries=1025), E_INVALID),
    (dict(temperature=0.0), E_INVALID), (dict(temperature=-1.0), E_INVALID),
    (dict(temperature=float("nan")), E_INVALID),
    (dict(temperature=float("inf")), E_INVALID),
    (dict(temperature=1e-45), E_INVALID), (dict(logits=A + 2), E_INVALID),
    (dict(count=0, logits=None, losses=None, grad=None), 0)])
def test_distill_refusals(mgpu, grad_too, change, code):
    assert distill(mgpu.load_library(), grad_too, **change) == code


@pytest.mark.parametrize("change", [
    dict(grad=None), dict(grad_stride=99), dict(grad=A + 4),
    dict(grad=A, grad_stride=128), dict(grad=(1 << 30) + 2),
    dict(weights=C + 2)])
def test_distill_gradient_refusals(mgpu, change):
    assert distill(mgpu.load_library(), True, **change) == E_INVALID


def sample(lib, dtype=F32, logits=A, stride=100, count=2, vocab=100, uniforms=B,
           temperature=1.0, ts=None, k=0, ks=None, p=1.0, ps=None, m=0.0,
           ms=None, out=C):
    return lib.mgpu_b200_sample_tokens(dtype, logits, stride, count, vocab,
                                       uniforms, temperature, ts, k, ks, p, ps,
                                       m, ms, out, None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=F64), E_UNSUPPORTED), (dict(logits=None), E_INVALID),
    (dict(uniforms=None), E_INVALID), (dict(out=None), E_INVALID),
    (dict(stride=99), E_INVALID), (dict(count=-1), E_INVALID),
    (dict(temperature=-1.0), E_INVALID),
    (dict(temperature=float("nan")), E_INVALID), (dict(p=-0.5), E_INVALID),
    (dict(m=1.5), E_INVALID), (dict(m=-0.1), E_INVALID),
    (dict(p=float("nan")), E_INVALID), (dict(ts=B + 1), E_INVALID),
    (dict(ks=B + 1), E_INVALID),
    (dict(count=0, logits=None, uniforms=None, out=None), 0)])
def test_sample_refusals(mgpu, change, code):
    assert sample(mgpu.load_library(), **change) == code


def test_cpu_tensors_are_refused(mgpu):
    x = torch.zeros(2, 4)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: mgpu.embedding_lookup(x, i),
                 lambda: mgpu.embedding_gradient(x, i, 8),
                 lambda: mgpu.distill_loss(x, i[:, None], x[:, :1]),
                 lambda: mgpu.distill_loss_gradient(x, i[:, None], x[:, :1]),
                 lambda: mgpu.sample_tokens(x, x[:, 0])):
        with pytest.raises(TypeError):
            call()


def test_reference_gradient_of_the_loss_against_differences():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 40, generator=g).double()
    ids = torch.tensor([[1, 5, 5, -1], [0, 39, 2, 3], [-1, -1, -1, -1]])
    t = torch.randn(3, 4, generator=g)
    w = torch.tensor([0.5, 2.0, 1.0])
    d = torch.randn(3, 40, generator=g).double()

    def loss(z):
        # float64 logits go through `distill` unrounded; only the bounds use
        # the type.
        n, s = z.shape[0], 0.0
        for i in range(n):
            s += float(w[i]) * _loss64(z[i].numpy(), ids[i].numpy(),
                                       t[i].numpy(), 1.5)
        return s

    _, grad, _, _ = ref.distill(x.float(), ids, t, w, 1.5)
    z = x.float().double()
    h = 1e-5
    difference = (loss(z + h * d) - loss(z - h * d)) / (2 * h)
    # Central differences: h^2 times a third derivative of order 1, and
    # 1e-16 / h of rounding.
    assert abs(difference - float((torch.from_numpy(grad) * d).sum())) < 1e-8


def _loss64(x, ids, t, T):
    used = ids >= 0
    if not used.any():
        return 0.0
    p = np.exp(t[used].astype(np.float64) / T)
    p /= p.sum()
    log_q = x / T - np.log(np.exp(x / T).sum())
    return T * T * float((p * (np.log(p) - log_q[ids[used]])).sum())


def test_reference_sampling_by_hand():
    # Weights 1, 1/2, 1/4, 1/4 at the places 2, 0, 1, 3.
    x = np.log([0.5, 0.25, 1.0, 0.25])
    assert ref.sample_row(x, 0.0) == 0
    assert ref.sample_row(x, 0.24) == 0 and ref.sample_row(x, 0.26) == 1
    assert ref.sample_row(x, 0.5) == 2 and ref.sample_row(x, 0.9) == 3
    assert ref.sample_row(x, 0.0, top_k=1) == 2
    assert ref.sample_row(x, 0.999, top_k=3) == 2    # of the equal ones, 1
    assert ref.sample_row(x, 0.0, top_k=3) == 0
    assert ref.sample_row(x, 0.0, top_p=0.4) == 2
    assert ref.sample_row(x, 0.0, top_p=0.6) == 0
    assert ref.sample_row(x, 0.0, min_p=0.6) == 2
    assert ref.sample_row(x, 0.7, temperature=0.0) == 2
    assert ref.sample_row([-np.inf, np.nan], 0.5) == -1
    assert ref.sample_row([-np.inf, -np.inf], 0.5) == -1
    assert ref.sample_row([1.0, np.inf, np.inf], 0.6) == 2


def test_ctypes_signatures_match_the_header(mgpu):
    lib = mgpu.load_library()
    assert lib.mgpu_b200_sample_tokens.argtypes[6] is ctypes.c_float
    assert len(lib.mgpu_b200_distill_loss_gradient.argtypes) == 16
