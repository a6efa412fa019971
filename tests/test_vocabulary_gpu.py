"""Embedding lookup and gradient, distillation and sampling on the GPU against
their definitions in 64 bits (vocabulary_reference.py, which also derives the
tolerances). Sampled tokens have to be equal."""
import math
import os
import subprocess

import numpy as np
import pytest
import torch

import vocabulary_reference as ref

pytestmark = pytest.mark.gpu

REALS = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def tokens_of(g, count, rows, dtype=torch.int64):
    """Falling off as one over the rank, some of them outside of the table."""
    u = torch.rand(count, device="cuda", generator=g)
    t = (torch.exp(u * math.log(rows + 1)) - 1).long().clamp(0, rows - 1)
    t[::13] = -1
    t[5::29] = rows
    return t.to(dtype)


def strided(x, extra, offset=0):
    """The same matrix inside a wider one, `offset` elements behind its start:
    other strides and alignments."""
    n, w = x.shape
    flat = torch.full((n * (w + extra) + offset,), 7.0, device="cuda",
                      dtype=x.dtype)
    view = flat[offset:].view(n, w + extra)[:, :w]
    view.copy_(x)
    return view


def close(got, want, bound):
    got = got.double().cpu()
    wrong = ~((got - want).abs() <= bound) & ~(got == want)
    assert not wrong.any(), "worst ratio %g at %s" % (
        float(((got - want).abs() / bound)[wrong].max()),
        torch.nonzero(wrong)[0].tolist())


# --- lookup ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
@pytest.mark.parametrize("width", [1, 3, 8, 64, 130, 1021, 4096, 9000])
def test_lookup(mgpu, dtype, ids, width):
    g = gen(width)
    table = randn(g, 77, width, dtype=dtype)
    tokens = tokens_of(g, 301, 77, ids)
    got = mgpu.embedding_lookup(table, tokens, scale=1.7)
    # The scale is a 32-bit number.
    want = ref.lookup(table, tokens, float(np.float32(1.7)))
    close(got, want, ref.lookup_bound(want, dtype))


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("extra,offset", [(1, 0), (8, 0), (8, 1), (5, 3), (2, 2)])
def test_lookup_strides_and_alignments(mgpu, dtype, extra, offset):
    g = gen(1)
    table = strided(randn(g, 40, 48, dtype=dtype), extra, offset)
    tokens = tokens_of(g, 90, 40)
    out = torch.empty(90 * 48 + 1, device="cuda", dtype=dtype)[
        offset % 2:][:90 * 48].view(90, 48)
    assert mgpu.embedding_lookup(table, tokens, out=out) is out
    want = ref.lookup(table, tokens, 1.0)
    close(out, want, ref.lookup_bound(want, dtype))


def test_lookup_shapes_and_far_tokens(mgpu):
    g = gen(2)
    table = randn(g, 10, 16)
    tokens = torch.tensor([[0, 9, -1], [10, 2**40, -2**63]], device="cuda")
    got = mgpu.embedding_lookup(table, tokens)
    assert got.shape == (2, 3, 16)
    assert torch.equal(got[0, :2], table[[0, 9]])
    assert not got[0, 2].any() and not got[1].any()
    assert mgpu.embedding_lookup(table, tokens[:0]).shape == (0, 3, 16)
    assert not mgpu.embedding_lookup(table[:0], tokens).any()
    one = torch.tensor(3, device="cuda", dtype=torch.int32)
    assert torch.equal(mgpu.embedding_lookup(table, one), table[3])


def test_lookup_infinities_stay_in_their_rows(mgpu):
    table = torch.full((3, 32), float("nan"), device="cuda")
    table[1] = 1.0
    tokens = torch.tensor([1, -1, 0, 1], device="cuda")
    got = mgpu.embedding_lookup(table, tokens, scale=0.5)
    assert torch.equal(got[0], got[3]) and (got[0] == 0.5).all()
    assert not got[1].any() and got[2].isnan().all()


def test_lookup_beyond_32_bit_offsets(mgpu):
    """A table of 2^31 + 2^20 elements: rows behind the 32-bit border."""
    width = 2048
    rows = (1 << 20) + 512
    table = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    marks = torch.tensor([0, 1 << 19, (1 << 20) - 1, 1 << 20, rows - 1],
                         device="cuda")
    table[marks] = randn(gen(3), 5, width, dtype=torch.bfloat16)
    assert torch.equal(mgpu.embedding_lookup(table, marks), table[marks])


# --- gradient ------------------------------------------------------------------

def check_gradient(mgpu, grad, tokens, rows, scale=1.0, out_dtype=None,
                   accumulate=False):
    out_dtype = out_dtype or grad.dtype
    start = None
    out = torch.full((rows, grad.shape[-1]), float("nan"), device="cuda",
                     dtype=out_dtype)
    if accumulate:
        start = randn(gen(99), rows, grad.shape[-1], dtype=out_dtype)
        out.copy_(start)
    got = mgpu.embedding_gradient(grad, tokens, rows, scale=scale, out=out,
                                  accumulate=accumulate)
    assert got is out
    want, size, times = ref.gradient(grad, tokens, rows,
                                     float(np.float32(scale)), start)
    close(out, want, ref.gradient_bound(want, size, times, out_dtype, start))
    if accumulate:
        untouched = (times == 0).to("cuda")
        assert torch.equal(out[untouched], start[untouched])
    return out


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype,out_dtype", [
    (torch.float32, torch.float32), (torch.float16, torch.float16),
    (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
    (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("count,rows,width", [
    (1, 1, 1), (1, 300, 64), (63, 5, 8), (64, 64, 130), (65, 1000, 33),
    (4096, 100, 16), (4097, 511, 40), (9001, 513, 8), (700, 3000, 2056)])
def test_gradient(mgpu, count, rows, width, dtype, out_dtype, accumulate):
    g = gen(count + width)
    grad = randn(g, count, width, dtype=dtype)
    tokens = tokens_of(g, count, rows,
                       torch.int32 if count % 2 else torch.int64)
    check_gradient(mgpu, grad, tokens, rows, 0.37, out_dtype, accumulate)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("kind", ["same", "two", "none", "first", "last",
                                  "falling", "runs_of_64", "each"])
def test_gradient_shapes_of_runs(mgpu, kind, accumulate):
    """Runs that fill tiles, end on their borders, or are missing."""
    count, rows, width = 1000, 2000, 24
    t = torch.arange(count, device="cuda")
    tokens = {"same": t * 0 + 777, "two": (t % 2) * 1999, "none": t * 0 - 1,
              "first": t * 0, "last": t * 0 + 1999, "falling": 1999 - t,
              "runs_of_64": t // 64, "each": t * 2}[kind]
    grad = randn(gen(4), count, width)
    check_gradient(mgpu, grad, tokens, rows, 1.0, None, accumulate)


@pytest.mark.parametrize("rows", [1, 2, 255, 256, 511, 512, 513, 4095, 4096,
                                  262143, 262144, 300000])
def test_gradient_numbers_of_rows(mgpu, rows):
    """Around the digits of the sort: one to three passes."""
    g = gen(rows)
    tokens = torch.randint(0, rows, (3000,), device="cuda", generator=g)
    tokens[:4] = torch.tensor([rows - 1, rows, -1, 0], device="cuda")
    check_gradient(mgpu, randn(g, 3000, 4), tokens, rows)


def test_gradient_of_nothing(mgpu):
    grad = torch.zeros(0, 8, device="cuda")
    tokens = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert not mgpu.embedding_gradient(grad, tokens, 100).any()
    out = torch.ones(100, 8, device="cuda")
    mgpu.embedding_gradient(grad, tokens, 100, out=out, accumulate=True)
    assert (out == 1).all()
    assert mgpu.embedding_gradient(grad, tokens, 0).shape == (0, 8)


@pytest.mark.parametrize("count", [0, 1, 5000, 140000])
def test_gradient_leaves_a_status_in_its_workspace(mgpu, count):
    """The word that workspace_status reads, here in a workspace full of ones,
    and in the stream's own between calls that share it."""
    g = gen(count)
    tokens = tokens_of(g, count, 3000)
    grad = randn(g, count, 8)
    need = mgpu.load_library().mgpu_b200_embedding_gradient_workspace_bytes(
        count, 3000, 8, 0)
    workspace = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    want = mgpu.embedding_gradient(grad, tokens, 3000, workspace=workspace)
    assert mgpu.workspace_status(workspace) == 0
    assert torch.equal(mgpu.embedding_gradient(grad, tokens, 3000), want)
    assert mgpu.workspace_status() == 0
    x = torch.arange(1000, dtype=torch.int32, device="cuda")
    assert torch.equal(mgpu.scan(x, inclusive=True), torch.cumsum(x, 0).int())
    assert mgpu.workspace_status() == 0


def test_gradient_leaves_out_padding_whatever_it_holds(mgpu):
    grad = randn(gen(5), 200, 64)
    tokens = tokens_of(gen(5), 200, 50)
    outside = (tokens < 0) | (tokens >= 50)
    want = mgpu.embedding_gradient(grad, tokens, 50)
    grad[outside] = float("nan")
    assert torch.equal(mgpu.embedding_gradient(grad, tokens, 50), want)


@pytest.mark.parametrize("extra,offset", [(1, 0), (8, 0), (8, 1), (4, 2)])
@pytest.mark.parametrize("dtype", REALS)
def test_gradient_strides(mgpu, dtype, extra, offset):
    g = gen(6)
    grad = strided(randn(g, 500, 72, dtype=dtype), extra, offset)
    check_gradient(mgpu, grad, tokens_of(g, 500, 90), 90,
                   out_dtype=torch.float32)


def test_gradient_into_an_output_of_8_byte_alignment(mgpu):
    g = gen(7)
    grad = randn(g, 300, 64, dtype=torch.bfloat16)
    tokens = tokens_of(g, 300, 40)
    out = torch.zeros(40 * 64 + 2, device="cuda")[2:].view(40, 64)
    mgpu.embedding_gradient(grad, tokens, 40, out=out)
    want, size, times = ref.gradient(grad, tokens, 40, 1.0)
    close(out, want, ref.gradient_bound(want, size, times, torch.float32))


def test_gradient_is_the_same_every_time(mgpu):
    g = gen(8)
    grad = randn(g, 20000, 96)
    tokens = tokens_of(g, 20000, 5000)
    first = mgpu.embedding_gradient(grad, tokens, 5000)
    for _ in range(5):
        assert torch.equal(mgpu.embedding_gradient(grad, tokens, 5000), first)


def test_gradient_of_many_positions(mgpu):
    """70,001 positions with one token for a third of them."""
    g = gen(9)
    tokens = tokens_of(g, 70001, 30011)
    tokens[::3] = 12345
    check_gradient(mgpu, randn(g, 70001, 40, dtype=torch.bfloat16), tokens,
                   30011, out_dtype=torch.float32)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("count,rows", [(32769, 900), (131072, 511),
                                        (131073, 70000), (300001, 300000)])
def test_gradient_of_each_form_of_the_sort(mgpu, count, rows, accumulate):
    """Around the numbers of positions that one cluster takes."""
    g = gen(count)
    check_gradient(mgpu, randn(g, count, 12), tokens_of(g, count, rows), rows,
                   accumulate=accumulate)


def test_gradient_against_differences_of_the_lookup(mgpu):
    """The lookup is linear: <lookup(d), grad> = <d, gradient(grad)>."""
    g = gen(10)
    d = randn(g, 211, 72)
    tokens = tokens_of(g, 900, 211).view(30, 30)
    grad = randn(g, 30, 30, 72)
    there = mgpu.embedding_lookup(d, tokens, scale=1.5).double()
    back = mgpu.embedding_gradient(grad, tokens, 211, scale=1.5).double()
    a = float((there * grad.double()).sum())
    b = float((back * d.double()).sum())
    size = float((there * grad.double()).abs().sum())
    # Each product carries a rounding of the lookup, and each gradient at most
    # 901 of its sum's terms.
    assert abs(a - b) <= 2.0 ** -24 * 905 * size


# --- distillation ----------------------------------------------------------------

def teacher_of(g, count, vocab, entries, ids=torch.int64, dtype=torch.float32):
    at = torch.randint(0, vocab, (count, entries), device="cuda", generator=g)
    at[::5, entries // 2:] = -1
    at[1::6] = -1
    at[2::7, 0] = vocab
    return at.to(ids), (randn(g, count, entries) * 3).to(dtype)


def check_distill(mgpu, logits, at, teacher, weights=None, T=1.0, out=None):
    want, grad, loss_bound, grad_bound = (
        torch.from_numpy(x) for x in ref.distill(logits, at, teacher, weights, T))
    plain = ref.distill(logits, at, teacher, None, T)
    close(mgpu.distill_loss(logits, at, teacher, temperature=T),
          torch.from_numpy(plain[0]), torch.from_numpy(plain[2]))
    loss, got = mgpu.distill_loss_gradient(
        logits, at, teacher, row_weights=weights, temperature=T, out=out)
    close(loss, want, loss_bound)
    close(got, grad, grad_bound)
    return loss, got


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("count,vocab,entries,T", [
    (1, 1, 1, 1.0), (3, 2, 5, 0.5), (9, 100, 1, 2.0), (30, 1000, 7, 1.0),
    (17, 4099, 64, 1.0), (8, 8192, 300, 4.0), (5, 50021, 33, 0.7),
    (2, 16384, 1024, 1.0)])
def test_distill(mgpu, count, vocab, entries, T, dtype):
    g = gen(vocab + entries)
    logits = randn(g, count, vocab, dtype=torch.float32) * 4
    at, teacher = teacher_of(g, count, vocab, entries,
                             torch.int32 if count % 2 else torch.int64,
                             REALS[entries % 3])
    weights = torch.rand(count, device="cuda", generator=g)
    weights[3::4] = 0
    check_distill(mgpu, logits.to(dtype), at, teacher, weights, T)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_of_few_rows_of_a_large_vocabulary(mgpu, dtype):
    g = gen(11)
    for count in (1, 3):
        logits = (randn(g, count, 131072) * 3).to(dtype)
        at = torch.randint(0, 131072, (count, 100), device="cuda", generator=g)
        check_distill(mgpu, logits, at, randn(g, count, 100) * 2)


def test_distill_the_same_token_twice(mgpu):
    g = gen(12)
    logits = randn(g, 4, 64)
    at = torch.tensor([[3, 3, 3, 9], [9, 3, 9, 3], [0, 0, 0, 0],
                       [63, -1, 63, 62]], device="cuda")
    check_distill(mgpu, logits, at, randn(g, 4, 4))


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("extra,offset", [(1, 0), (8, 0), (8, 1), (24, 2)])
def test_distill_strides_and_in_place(mgpu, dtype, extra, offset):
    g = gen(13)
    x = (randn(g, 6, 1000) * 3).to(dtype)
    at, teacher = teacher_of(g, 6, 1000, 10)
    logits = strided(x, extra, offset)
    _, apart = check_distill(mgpu, logits, at, teacher,
                             out=strided(x * 0, extra + 8, offset))
    around = logits.as_strided((6, 1000 + extra), logits.stride(),
                               logits.storage_offset()) if not offset else None
    loss, same = mgpu.distill_loss_gradient(logits, at, teacher, out=logits)
    assert same is logits and torch.equal(same, apart)
    if around is not None:                # what lies between the rows stays
        assert (around[:, 1000:] == 7).all()


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("vocab", [1, 7, 1000, 33001])
def test_distill_gradient_aligned_apart_from_the_logits(mgpu, dtype, vocab):
    g = gen(19)
    x = (randn(g, 5, vocab) * 3).to(dtype)
    at, teacher = teacher_of(g, 5, vocab, 40)
    weights = torch.tensor([1.0, 0.5, 0.0, 2.0, 1.0], device="cuda")
    x[4] = -float("inf")
    check_distill(mgpu, strided(x, 3), at, teacher, weights,
                  out=strided(x * 0, 3, 1))
    check_distill(mgpu, strided(x, 1), at, teacher, weights,
                  out=strided(x * 0, 2))


@pytest.mark.parametrize("grad_rows", [1, 40, 700])
@pytest.mark.parametrize("vocab", [5, 3000, 60000, 140001])
def test_distill_numbers_of_rows(mgpu, grad_rows, vocab):
    """Rows that stay with their CTAs for several rounds, in clusters of every
    size; a sample of them is compared."""
    g = gen(vocab)
    logits = (randn(g, grad_rows, vocab) * 3).bfloat16()
    at, teacher = teacher_of(g, grad_rows, vocab, 20)
    loss, grad = mgpu.distill_loss_gradient(logits, at, teacher)
    rows = sorted({0, grad_rows // 2, grad_rows - 1})
    want, slope, loss_bound, grad_bound = (torch.from_numpy(v) for v in
        ref.distill(logits[rows], at[rows], teacher[rows], None, 1.0))
    close(loss[rows], want, loss_bound)
    close(grad[rows], slope, grad_bound)
    assert torch.equal(loss, mgpu.distill_loss(logits, at, teacher))
    # Every row by itself: the loss from the gradient's own probabilities.
    few = (at >= 0) & (at < vocab)
    p = torch.softmax(torch.where(few, teacher, -float("inf")).double(), 1)
    p = torch.nan_to_num(p)
    log_q = torch.log_softmax(logits.double(), 1)
    plain = torch.special.entr(p).sum(1).neg() - (
        p * log_q.gather(1, at.clamp(0, vocab - 1))).sum(1)
    # 32-bit sums of `vocab` weights, and of 20 products of order 30.
    assert torch.allclose(loss.double(), plain, rtol=1e-4, atol=1e-4)
    assert grad.float().sum(1).abs().max() <= 2.0 ** -8 * 2.01


@pytest.mark.parametrize("count,vocab,dtype", [
    (600, 131072, torch.bfloat16), (509, 50021, torch.float32),
    (2048, 32768, torch.float16)])
def test_distill_is_the_same_every_time(mgpu, count, vocab, dtype):
    """Bit for bit: a buffer that is filled again before it has been read would
    show."""
    g = gen(20)
    x = (randn(g, count, vocab) * 3).to(dtype)
    at, teacher = teacher_of(g, count, vocab, 64)
    loss, grad = mgpu.distill_loss_gradient(x, at, teacher)
    for _ in range(25):
        again = mgpu.distill_loss_gradient(x, at, teacher)
        assert torch.equal(again[0], loss) and torch.equal(again[1], grad)
    same = mgpu.distill_loss_gradient(x, at, teacher, out=x)
    assert torch.equal(same[1], grad) and torch.equal(same[0], loss)


def test_distill_rows_without_a_distribution(mgpu):
    inf = float("inf")
    x = torch.randn(7, 300, device="cuda", generator=gen(14))
    at = torch.arange(4, device="cuda").repeat(7, 1) * 70
    teacher = torch.randn(7, 4, device="cuda", generator=gen(15))
    weights = torch.ones(7, device="cuda")
    at[0] = -1                             # no teacher
    teacher[1] = -inf                      # no teacher either
    x[2] = -inf                            # no student
    weights[3] = 0                         # masked, whatever it holds
    x[3] = float("nan")
    x[4, 1:] = -inf                        # one token is left
    at[4] = torch.tensor([0, -1, -1, -1], device="cuda")
    x[5, 70] = -inf                        # the teacher wants what cannot be
    loss, grad = mgpu.distill_loss_gradient(x, at, teacher, weights)
    for row in range(4):
        assert loss[row] == 0 and not grad[row].any()
    assert loss[4] == 0 and not grad[4].any()
    assert loss[5] == inf and grad[5].isfinite().all() and grad[5, 70] < 0
    want = ref.distill(x[6:], at[6:], teacher[6:], None, 1.0)
    assert abs(float(loss[6]) - want[0][0]) <= want[2][0]
    plain = mgpu.distill_loss(x, at, teacher)
    assert plain[3].isnan() and torch.equal(plain[4:], loss[4:])


def test_distill_masks_of_the_lowest_value_and_wrong_numbers(mgpu):
    g = gen(16)
    for dtype in REALS:
        x = randn(g, 3, 2000, dtype=dtype)
        x[:, 100:1900] = torch.finfo(dtype).min
        at, teacher = (torch.tensor([[5, 1950, 20]] * 3, device="cuda"),
                       randn(g, 3, 3))
        check_distill(mgpu, x, at, teacher)
        x[0, 500] = float("nan")
        x[1, 500] = float("inf")
        loss, grad = mgpu.distill_loss_gradient(x, at, teacher)
        assert loss[0].isnan() and loss[1].isnan() and loss[2].isfinite()
        assert grad[0].isnan().any() and grad[2].isfinite().all()


def test_distill_masked_entries_of_the_teacher(mgpu):
    """An entry of -infinity has no part; the others' stay as they are."""
    g = gen(17)
    x, at = randn(g, 2, 500), torch.tensor([[1, 2, 3]] * 2, device="cuda")
    t = randn(g, 2, 3)
    t[:, 1] = -float("inf")
    full = mgpu.distill_loss_gradient(x, at, t)
    less = mgpu.distill_loss_gradient(x, at[:, ::2].contiguous(),
                                      t[:, ::2].contiguous())
    assert torch.equal(full[0], less[0]) and torch.equal(full[1], less[1])


def test_distill_without_entries(mgpu):
    x = torch.randn(3, 50, device="cuda")
    loss, grad = mgpu.distill_loss_gradient(
        x, torch.zeros(3, 0, dtype=torch.int32, device="cuda"),
        torch.zeros(3, 0, device="cuda"))
    assert not loss.any() and not grad.any()


def test_distill_gradient_against_differences(mgpu):
    """Along a direction d: central differences of the 64-bit loss at the
    32-bit logits."""
    g = gen(18)
    x = randn(g, 5, 700) * 2
    at, teacher = teacher_of(g, 5, 700, 12)
    _, grad = mgpu.distill_loss_gradient(x, at, teacher, temperature=2.0)
    d = randn(g, 5, 700).double()
    h = 1e-4

    def loss(z):
        return ref.distill(z, at, teacher, None, 2.0)[0].sum()

    up, down = ((x.double() + s * h * d) for s in (1, -1))
    difference = (loss(up) - loss(down)) / (2 * h)
    _, _, _, bound = ref.distill(x, at, teacher, None, 2.0)
    slack = float((torch.from_numpy(bound) * d.abs().cpu()).sum())
    # h^2 / 6 of a third derivative: at most sum |d|^3 q (1/T) per row.
    curve = h * h * float((d.abs() ** 3).amax()) * 5
    assert abs(difference - float((grad.double() * d).sum())) <= slack + curve \
        + 1e-10


# --- sampling ----------------------------------------------------------------------

SETTINGS = [
    dict(), dict(temperature=0.0), dict(temperature=0.3), dict(temperature=7.0),
    dict(top_k=1), dict(top_k=5), dict(top_k=700), dict(top_p=0.0),
    dict(top_p=0.5), dict(top_p=0.999), dict(min_p=0.2), dict(min_p=1.0),
    dict(top_k=40, top_p=0.8, min_p=0.05, temperature=0.7),
    dict(top_k=5000, top_p=0.9), dict(top_p=0.3, min_p=0.001, temperature=2.0)]


def check_sample(mgpu, logits, seed=0, uniform=None, **settings):
    if uniform is None:
        uniform = torch.rand(logits.shape[0], device="cuda",
                             generator=gen(seed))
    got = mgpu.sample_tokens(logits, uniform, **settings).cpu()
    want = ref.sample(logits, uniform, **settings)
    assert torch.equal(got, want), (got[got != want], want[got != want])
    return got


def sharp(g, count, vocab, dtype):
    """Rows from flat to nearly certain."""
    x = randn(g, count, vocab) * 2.5
    strong = (torch.rand(count, 9, device="cuda", generator=g) * vocab).long()
    x.scatter_add_(1, strong, torch.linspace(0, 14, count, device="cuda")[
        :, None] + torch.rand(count, 9, device="cuda", generator=g) * 3)
    return x.to(dtype)


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 4099, 33000])
def test_sample(mgpu, vocab, dtype, settings):
    check_sample(mgpu, sharp(gen(vocab), 24, vocab, dtype), vocab, **settings)


@pytest.mark.parametrize("settings", SETTINGS[::3] + [SETTINGS[12]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_large_vocabulary(mgpu, dtype, settings):
    check_sample(mgpu, sharp(gen(20), 7, 131072, dtype), 5, **settings)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=37), dict(top_p=0.51),
                                      dict(top_k=900, top_p=0.5),
                                      dict(min_p=0.5)])
@pytest.mark.parametrize("kinds", [1, 2, 5])
def test_sample_equal_logits(mgpu, kinds, settings):
    """All equal, and a few values that very many tokens share: the lowest
    indices are kept."""
    g = gen(21)
    x = torch.randint(0, kinds, (40, 3001), device="cuda", generator=g).float()
    check_sample(mgpu, x, 1, **settings)
    check_sample(mgpu, x.bfloat16(), 1, **settings)


def test_sample_signed_zeros_are_equal(mgpu):
    x = torch.zeros(8, 64, device="cuda")
    x[:, ::2] = -0.0
    u = torch.arange(8, device="cuda") / 8
    got = check_sample(mgpu, x, uniform=u, top_k=8)
    assert got.tolist() == list(range(8))


def test_sample_borders_of_the_given_numbers(mgpu):
    """Equal weights: u = j / n belongs to token j; 0 to the first token of
    weight, the greatest number below 1 to the last."""
    n = 4096
    x = torch.full((n, n), -2.5, device="cuda")
    u = torch.arange(n, device="cuda", dtype=torch.float32) / n
    got = mgpu.sample_tokens(x, u)
    assert torch.equal(got, torch.arange(n, device="cuda", dtype=torch.int32))
    x[:, :7] = -float("inf")
    x[:, 4000:] = -float("inf")
    u[0], u[1], u[2] = 0.0, 1 - 2.0 ** -24, 1.0
    got = mgpu.sample_tokens(x, u)
    assert got[0] == 7 and got[1] == 3999 and got[2] == 3999


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("settings", [dict(), dict(top_k=50), dict(top_p=0.9),
                                      dict(temperature=0.0), dict(min_p=0.1)])
def test_sample_masks(mgpu, dtype, settings):
    """-infinity and the type's lowest value in masked places, rows with one
    token, rows with none, rows with a NaN."""
    x = sharp(gen(22), 12, 5000, dtype)
    x[0, 100:] = -float("inf")
    x[1, :4999] = -float("inf")
    x[2] = -float("inf")
    x[3, 4321] = float("nan")
    x[4, 5:] = torch.finfo(dtype).min
    x[5] = torch.finfo(dtype).min
    x[6, 17] = x[6, 400] = float("inf")
    got = check_sample(mgpu, x, 3, **settings)
    assert got[1] == 4999 and got[2] == -1 and got[3] == -1


@pytest.mark.parametrize("dtype", REALS)
def test_sample_top_k_of_unlike_parts(mgpu, dtype):
    """The greatest tokens in one part of the row, spread over all, equal, far
    apart, large against their distances, and infinite."""
    x = randn(gen(30), 10, 40000, dtype=dtype)
    x[0, 39000:39100] = 30.0
    x[1, ::400] = 12.0
    x[2] = 0.0
    x[3] = torch.arange(40000, device="cuda") % 977 / 8
    x[4] = 3e4 + torch.arange(40000, device="cuda") % 50
    x[5, 7::5000] = float("inf")
    x[6, :20000] = -float("inf")
    x[7] = -float("inf")
    x[7, 5::9000] = 1.0
    x[8, 100:200] = float("inf")
    for k in (1, 3, 50, 64, 200):
        for t in (1.0, 0.01, 100.0):
            check_sample(mgpu, x, k, top_k=k, temperature=t)


def test_sample_top_k_beyond_the_tokens_left(mgpu):
    x = torch.full((4, 3000), -float("inf"), device="cuda")
    x[:, 2000:2005] = torch.randn(4, 5, device="cuda", generator=gen(23))
    got = check_sample(mgpu, x, top_k=50, top_p=0.99)
    assert ((got >= 2000) & (got < 2005)).all()


def test_sample_settings_by_row(mgpu):
    g = gen(24)
    n, vocab = 64, 9001
    pick = torch.arange(n, device="cuda")
    check_sample(
        mgpu, sharp(g, n, vocab, torch.float32), 7,
        temperature=torch.where(pick % 7 == 0, 0.0, 0.2 + pick / 20.0),
        top_k=torch.where(pick % 3 == 0, pick * 4, 0).int(),
        top_p=torch.where(pick % 2 == 0, 0.3 + pick / 80.0, 1.0),
        min_p=torch.where(pick % 5 == 0, pick / 300.0, 0.0))


@pytest.mark.parametrize("extra,offset", [(1, 0), (7, 0), (8, 1), (5, 3)])
@pytest.mark.parametrize("dtype", REALS)
def test_sample_strides(mgpu, dtype, extra, offset):
    x = strided(sharp(gen(25), 10, 4000, dtype), extra, offset)
    check_sample(mgpu, x, 2, top_k=100, top_p=0.9)


@pytest.mark.parametrize("settings", [
    dict(temperature=3e38), dict(temperature=3e38, top_p=0.5),
    dict(temperature=1e-38), dict(temperature=1e-45, top_p=0.9),
    dict(temperature=1e30, top_k=3, min_p=0.5)])
def test_sample_far_temperatures(mgpu, settings):
    x = sharp(gen(27), 9, 3000, torch.float32)
    x[:, ::3] = -float("inf")
    check_sample(mgpu, x, 4, **settings)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("count,vocab", [(1, 300000), (3, 700001), (200, 9000),
                                         (40, 70001)])
def test_sample_parts_in_shared_memory_and_not(mgpu, dtype, count, vocab):
    """Rows of one CTA to eight, parts that stay in shared memory and others."""
    x = sharp(gen(28), count, vocab, dtype)
    for i, settings in enumerate([dict(top_p=0.9, min_p=0.001),
                                  dict(top_k=20), dict(top_k=3000, top_p=0.7)]):
        check_sample(mgpu, x, i, **settings)


def test_sample_nearly_all_of_the_weight(mgpu):
    """Borders far down, among tokens of next to no weight."""
    x = randn(gen(29), 12, 20000) * 6
    for p in (0.99999, 1 - 2.0 ** -24, 1e-7):
        check_sample(mgpu, x, 6, top_p=p)


def test_sample_many_rows(mgpu):
    x = sharp(gen(26), 3000, 257, torch.float16)
    check_sample(mgpu, x, 9, top_p=0.8)


# --- all of them together ------------------------------------------------------------

def training_step(mgpu, table, head, tokens, at, teacher, weights):
    """Lookup, a head, distillation, and the gradients back to the table."""
    scale = table.shape[1] ** 0.5
    hidden = mgpu.embedding_lookup(table, tokens, scale=scale)
    logits = hidden.view(-1, table.shape[1]) @ head
    loss, g = mgpu.distill_loss_gradient(logits, at, teacher, weights,
                                         temperature=2.0, out=logits)
    back = (g @ head.t()).view(hidden.shape)
    return loss, mgpu.embedding_gradient(back, tokens, table.shape[0],
                                         scale=scale)


def step_inputs():
    g = gen(30)
    table, head = randn(g, 800, 64), randn(g, 64, 1200) * 0.05
    tokens = tokens_of(g, 96, 800).view(4, 24)
    at, teacher = teacher_of(g, 96, 1200, 8)
    weights = (tokens.view(-1) >= 0).float() / 96
    return table, head, tokens, at, teacher, weights


def test_a_training_step_against_differences(mgpu):
    table, head, tokens, at, teacher, weights = step_inputs()
    _, grad = training_step(mgpu, table, head, tokens, at, teacher, weights)
    d = torch.zeros_like(table)
    live = tokens[(tokens >= 0) & (tokens < 800)].unique()
    d[live] = randn(gen(31), live.numel(), 64)
    h = 1e-4

    def loss(t):
        x = ref.lookup(t, tokens, 8.0).view(-1, 64) @ head.double().cpu()
        return float(np.sum(ref.distill(x, at, teacher, None, 2.0)[0]
                            * weights.double().cpu().numpy()))

    want = (loss(table.double() + h * d.double())
            - loss(table.double() - h * d.double())) / (2 * h)
    got = float((grad.double() * d.double()).sum())
    # 64-term products in 32 bits, thrice: the step's gradient is good to about
    # 3 * 64 * 2^-24 of the size of its terms (1e-5); differences to 1e-6.
    size = float((grad.double() * d.double()).abs().sum())
    assert abs(got - want) <= 2e-5 * size + 1e-6


def test_a_captured_training_step(mgpu):
    """Captured once, replayed with other inputs: what an eager step gives. Two
    graphs of one step that are replayed at the same time share nothing."""
    table, head, tokens, at, teacher, weights = step_inputs()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        training_step(mgpu, table, head, tokens, at, teacher, weights)
    torch.cuda.current_stream().wait_stream(side)
    graphs, results, inputs = [], [], []
    for i in range(2):
        mine = tokens.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(training_step(mgpu, table, head, mine, at, teacher,
                                         weights))
        graphs.append(graph)
        inputs.append(mine)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        new = [tokens_of(gen(40 + 2 * turn + i), 96, 800).view(4, 24)
               for i in range(2)]
        for mine, n in zip(inputs, new):
            mine.copy_(n)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (loss, grad), n in zip(results, new):
            want = training_step(mgpu, table, head, n, at, teacher, weights)
            assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])


def test_a_decode_loop(mgpu):
    """Lookup, head, sampling, and the token back into the lookup."""
    table, head, *_ = step_inputs()
    head = head[:, :800].contiguous()
    u = torch.rand(6, 5, device="cuda", generator=gen(33))
    token = torch.arange(5, device="cuda", dtype=torch.int32)
    for step in range(6):
        logits = mgpu.embedding_lookup(table, token, scale=8.0) @ head
        token = mgpu.sample_tokens(logits, u[step], temperature=0.9, top_k=40,
                                   top_p=0.95, min_p=0.01)
        want = ref.sample(logits, u[step], 0.9, 40, 0.95, 0.01)
        assert torch.equal(token.cpu(), want)


def test_calls_on_other_streams(mgpu):
    """Eight calls on eight streams at once, each with scratch of its own."""
    g = gen(34)
    work = [(randn(g, 5000, 64), tokens_of(g, 5000, 3000)) for _ in range(8)]
    want = [mgpu.embedding_gradient(a, t, 3000) for a, t in work]
    streams = [torch.cuda.Stream() for _ in range(8)]
    torch.cuda.synchronize()
    got = []
    for (a, t), s in zip(work, streams):
        with torch.cuda.stream(s):
            got.append(mgpu.embedding_gradient(a, t, 3000))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_refusals(mgpu):
    x = torch.randn(4, 32, device="cuda")
    i = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError):
        mgpu.embedding_lookup(x.double(), i)
    with pytest.raises(TypeError):
        mgpu.embedding_lookup(x, i.float())
    with pytest.raises(ValueError):
        mgpu.embedding_lookup(x.t(), i)
    with pytest.raises(ValueError):
        mgpu.embedding_lookup(x[:1].expand(4, 32), i)
    with pytest.raises(ValueError):
        mgpu.embedding_lookup(x, i, out=x[:3].contiguous())
    with pytest.raises(mgpu.MgpuError):
        mgpu.embedding_lookup(x, i, out=x)
    with pytest.raises(ValueError):
        mgpu.embedding_gradient(x, i[:3], 10)
    with pytest.raises(ValueError):
        mgpu.embedding_gradient(x, i, 10, accumulate=True)
    with pytest.raises(ValueError):
        mgpu.embedding_gradient(x, i, 2**32 + 5)
    with pytest.raises(TypeError):
        mgpu.embedding_gradient(x, i, 10, out=torch.zeros(
            10, 32, device="cuda", dtype=torch.float16))
    with pytest.raises(mgpu.MgpuError):
        mgpu.embedding_gradient(x, i, 4, workspace=torch.zeros(
            128, dtype=torch.uint8, device="cuda"))
    at = i[:, None]
    with pytest.raises(ValueError):
        mgpu.distill_loss(x, at, x[:, :2].contiguous())
    with pytest.raises(ValueError):
        mgpu.distill_loss(x, at[:3], x[:3, :1].contiguous())
    with pytest.raises(mgpu.MgpuError):
        mgpu.distill_loss(x, at, x[:, :1].contiguous(), temperature=0.0)
    with pytest.raises(ValueError):
        mgpu.distill_loss_gradient(x, at, x[:, :1].contiguous(),
                                   row_weights=x[:3, 0].contiguous())
    with pytest.raises(mgpu.MgpuError):
        many = torch.zeros(4, 1025, dtype=torch.int32, device="cuda")
        mgpu.distill_loss(x, many, many.float())
    big = torch.randn(4, 40, device="cuda")
    with pytest.raises(mgpu.MgpuError):
        mgpu.distill_loss_gradient(big[:, :32], at, x[:, :1].contiguous(),
                                   out=big[:, 8:])
    u = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError):
        mgpu.sample_tokens(x, u[:3])
    with pytest.raises(TypeError):
        mgpu.sample_tokens(x, u, top_k=u)
    with pytest.raises(ValueError):
        mgpu.sample_tokens(x, u, top_p=u[:2])
    with pytest.raises(mgpu.MgpuError):
        mgpu.sample_tokens(x, u, temperature=-1.0)
    for call in (lambda: mgpu.embedding_lookup([1], i),
                 lambda: mgpu.embedding_gradient(None, i, 4),
                 lambda: mgpu.distill_loss(3, at, x),
                 lambda: mgpu.sample_tokens("x", u)):
        with pytest.raises(TypeError):
            call()
    # More tokens than there are: all of them.
    assert torch.equal(mgpu.sample_tokens(x, u, top_k=2**40),
                       mgpu.sample_tokens(x, u))
    if torch.cuda.device_count() > 1:
        with pytest.raises(ValueError):
            mgpu.sample_tokens(x, u.to("cuda:1"))


def test_cpp_entry_points():
    """tests/cpp/test_vocabulary.cu: the templates on a context."""
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp",
                       "build", "test_vocabulary")
    if not os.path.exists(exe):
        pytest.fail("not built: run "
                    "python -c 'import __graft_entry__ as g; g.build()'")
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert "ALL PASSED" in run.stdout and not run.returncode, (
        run.stdout + run.stderr)
