"""The experts' products and their gradients against a plain implementation in 64 bits."""
from __future__ import annotations

import threading

import pytest

torch = pytest.importorskip("torch")

from libcusort_b200 import _capi, experts as X  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert X.product_status() == 0


def _few(x, w, g):
    return X.expert_products(x[:40], w, torch.tensor([20, 20], dtype=torch.int32, device="cuda"),
                             torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda"))


def _many(x, w, g):
    return X.expert_products(x, w, *plan([300, 500])[:2])


def _gradient(x, w, g):
    return X.expert_products_grad_weights(g, x, *plan([300, 500])[:2])


@pytest.mark.parametrize("skip", [0, 3, 13])
@pytest.mark.parametrize("call", [_few, _many, _gradient])
def test_a_wait_that_runs_out_is_told(call, skip):
    """Copies that never come: the kernel ends after a millisecond with a status, and the next call is right again."""
    x, w, g = (matrix(800, 1024, torch.bfloat16), weights_of(2, 1024, 2048, torch.bfloat16, "in_out"),
               matrix(800, 2048, torch.bfloat16, seed=4))
    right, lib = call(x, w, g), _capi.load()
    before = lib.cusort_set_wait_limit_ns(1_000_000)
    lib.cusort_debug_set_skip_tile(skip)
    try:
        call(x, w, g)
    finally:
        lib.cusort_debug_set_skip_tile(-1)
        lib.cusort_set_wait_limit_ns(before)
    told = X.product_status(), X.product_status()
    # every CTA has one tile at most here: of 1024 / 128 or 1024 / 64 steps, or of the segments' 300 and 500 rows by 64
    steps = {_few: 8, _many: 16, _gradient: 8}[call]
    assert told == ((1, 0) if skip < steps else (0, 0))
    assert torch.equal(call(x, w, g), right)


def test_results_and_weights_beyond_32_bits():
    c, o, capacity, _ = plan([400_000, 200_000])
    x, w = matrix(capacity, 64, torch.bfloat16), weights_of(2, 64, 4096, torch.bfloat16, "in_out")
    out = X.expert_products(x, w, c, o)  # 4.9 GB
    for at, e in ((slice(0, 50), 0), (slice(399_950, 400_000), 0), (slice(400_000, 400_050), 1),
                  (slice(capacity - 50, capacity), 1)):
        xe, we = x[at].double(), w[e].double()
        close(out[at], xe @ we, xe.abs() @ we.abs(), 64)
    del out, x, w
    counts = [0] * 540
    counts[0], counts[539] = 40, 70
    c, o, capacity, _ = plan(counts)
    x, g = matrix(capacity, 2048, torch.bfloat16), matrix(capacity, 2048, torch.bfloat16, seed=2)
    w = torch.zeros(540, 2048, 2048, dtype=torch.bfloat16, device="cuda")  # 4.5 GB
    w[0], w[539] = weights_of(2, 2048, 2048, torch.bfloat16, "in_out")
    out, grad = X.expert_products(x, w, c, o), X.expert_products_grad_weights(g, x, c, o)
    for at, e in ((slice(0, 40), 0), (slice(40, 110), 539)):
        xe, ge, we = x[at].double(), g[at].double(), w[e].double()
        close(out[at], xe @ we, xe.abs() @ we.abs(), 2048)
        close(grad[e], xe.T @ ge, xe.T.abs() @ ge.abs(), 70)
    assert not grad[1:539].any()


def plan(counts, align=1, tail=0):
    """counts, offsets, capacity and which rows belong to an expert."""
    offsets, at = [0], 0
    for c in counts:
        at += -(-c // align) * align
        offsets.append(at)
    there = torch.zeros(at + tail, dtype=torch.bool, device="cuda")
    for o, c in zip(offsets, counts):
        there[o:o + c] = True
    return (torch.tensor(counts, dtype=torch.int32, device="cuda"),
            torch.tensor(offsets, dtype=torch.int32, device="cuda"), at + tail, there)


def matrix(rows, width, dtype, there=None, pitch=None, shift=0, seed=0):
    """Random rows, NaN and infinities where ``there`` is false; rows `pitch` elements apart, `shift` behind a start."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pitch = pitch or width
    x = torch.randn(rows * pitch + shift + 8, generator=gen, device="cuda").to(dtype)[shift:].as_strided(
        (rows, width), (pitch, 1))
    if there is not None:
        x[~there] = torch.tensor([float("nan"), float("inf")], device="cuda").repeat(width)[:width].to(dtype)
    return x


def weights_of(experts, fin, fout, dtype, order, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (experts, fin, fout) if order == "in_out" else (experts, fout, fin)
    w = torch.randn(*shape, generator=gen, device="cuda").to(dtype)
    return w if order == "in_out" else w.transpose(1, 2)


def close(got, want, size, depth):
    """One rounding of the result (half a step: eps / 2 of it, and half the smallest subnormal), and `depth` 32-bit
    additions, each off by a step (2^-23) of at most the sum of all products' sizes."""
    info = torch.finfo(got.dtype)
    tiny = info.smallest_normal * info.eps / 2
    bound = info.eps / 2 * want.abs() + (1 + info.eps) * depth * 2.0 ** -23 * size + tiny
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4], want[bad][:4])


def check(counts, fin, fout, dtype="bf16", order="in_out", align=1, tail=0, pitch=None, shift=0, grad_pitch=None):
    dtype = TYPES[dtype]
    c, o, capacity, there = plan(counts, align, tail)
    x = matrix(capacity, fin, dtype, there, pitch, shift)
    g = matrix(capacity, fout, dtype, there, grad_pitch, seed=2)
    w = weights_of(len(counts), fin, fout, dtype, order)
    out = X.expert_products(x, w, c, o)
    grad_rows, grad_weights = X.expert_products_backward(g, x, w, c, o)
    assert out.shape == (capacity, fout) and out.dtype == dtype and out.is_contiguous()
    assert grad_rows.shape == x.shape and grad_weights.shape == w.shape
    assert grad_weights.stride() == w.stride() or min(fin, fout) == 1
    assert not out[~there].any() and not grad_rows[~there].any()
    for e, (first, count) in enumerate(zip(o.tolist(), counts)):
        at = slice(first, first + count)
        xe, ge, we = x[at].double(), g[at].double(), w[e].double()
        close(out[at], xe @ we, xe.abs() @ we.abs(), fin)
        close(grad_rows[at], ge @ we.T, ge.abs() @ we.T.abs(), fout)
        close(grad_weights[e], xe.T @ ge, xe.T.abs() @ ge.abs(), max(count, 1))


@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("fin,fout", [(64, 128), (128, 64), (72, 200), (8, 8), (512, 264), (200, 1032)])
def test_few_rows_an_expert(fin, fout, dtype, order):
    check([0, 1, 3, 0, 16, 17, 33, 64, 0, 40], fin, fout, dtype, order)


@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("counts", [[1], [3, 0, 5, 1, 0, 7], [0, 2, 0, 64], [1, 33, 0, 5, 0, 0, 1, 70]], ids=str)
@pytest.mark.parametrize("fin,fout", [(520, 136), (1032, 264), (2049, 200), (4096, 128)])
def test_few_tiles_with_a_long_contracted_dimension(fin, fout, counts, order):
    check(counts, fin, fout, "bf16", order)


@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("fin,fout", [(200, 4744), (1032, 9608), (64, 70)])
def test_sixteen_rows_at_most_over_wide_results(fin, fout, order):
    check([9, 0, 7], fin, fout, "bf16", order)
    check([16], fin, fout, "f16", order)


@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("fin,fout", [(64, 128), (264, 136), (136, 520)])
def test_many_rows_an_expert(fin, fout, dtype, order):
    check([0, 255, 1, 256, 257, 0, 300, 1000, 63, 65], fin, fout, dtype, order)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("align,tail", [(16, 0), (128, 70), (7, 1000), (1, 333)])
@pytest.mark.parametrize("fin,fout", [(64, 136), (40, 33)])
def test_rows_of_no_segment_are_zeros_and_not_read(fin, fout, align, tail, dtype):
    check([5, 0, 128, 130, 0, 1, 0], fin, fout, dtype, align=align, tail=tail)


@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("fin,fout", [(1, 1), (7, 5), (1, 64), (64, 1), (33, 130), (771, 257), (66, 72), (72, 66)])
def test_widths_of_no_16_bytes(fin, fout, order):
    check([3, 0, 70, 1, 20], fin, fout, "f16", order)
    check([3, 0, 70, 1, 20], fin, fout, "f32", order)


@pytest.mark.parametrize("pitch,shift,grad_pitch", [(80, 0, 72), (72, 4, 64), (65, 0, 67), (64, 8, 64), (64, 1, 71)])
def test_rows_apart_and_off_16_bytes(pitch, shift, grad_pitch):
    check([9, 130, 0, 31], 64, 64, "bf16", pitch=pitch, shift=shift, grad_pitch=grad_pitch)
    check([9, 130, 0, 31], 64, 64, "f32", pitch=pitch, shift=shift, grad_pitch=grad_pitch)


def test_one_expert_and_the_most():
    check([700], 136, 72)
    check([1], 64, 64)
    check([i % 3 for i in range(1024)], 64, 72)
    check([i % 3 for i in range(1024)], 24, 40, "f32")


def test_nothing_to_do():
    check([0, 0, 0], 64, 72)
    check([0, 0, 0], 64, 72, tail=50)
    check([0], 33, 5, "f16")
    check([0, 0, 0], 64, 72, "f32", tail=50)


def test_expanded_rows_and_weights():
    c, o, capacity, _ = plan([3, 5])
    x = matrix(1, 64, torch.bfloat16).expand(capacity, 64)
    w = weights_of(1, 64, 72, torch.bfloat16, "in_out").expand(2, 64, 72)
    close(X.expert_products(x, w, c, o), x.double() @ w[0].double(), x.double().abs() @ w[0].double().abs(), 64)


def test_weights_apart():
    c, o, capacity, _ = plan([30, 70])
    whole = weights_of(2, 80, 96, torch.bfloat16, "in_out")
    for w in (whole[:, :64, :72], whole[:, 3:67, 8:80], whole[:, :64, 1:73], whole.transpose(1, 2)[:, :64, 5:77]):
        x = matrix(capacity, 64, torch.bfloat16)
        out = X.expert_products(x, w, c, o)
        for e, at in enumerate((slice(0, 30), slice(30, 100))):
            close(out[at], x[at].double() @ w[e].double(), x[at].double().abs() @ w[e].double().abs(), 64)


def test_infinities_and_nan_stay_in_their_rows():
    c, o, capacity, _ = plan([40, 40])
    x = matrix(capacity, 128, torch.bfloat16)
    w = weights_of(2, 128, 128, torch.bfloat16, "in_out")
    clean = X.expert_products(x, w, c, o)
    x[7, 3], x[50, 100], x[39, 0] = float("nan"), float("inf"), float("-inf")
    out = X.expert_products(x, w, c, o)
    hit = torch.zeros(capacity, dtype=torch.bool, device="cuda")
    hit[[7, 39, 50]] = True
    assert torch.equal(out[~hit], clean[~hit]) and not torch.isfinite(out[hit]).any()


def test_overflow_of_the_type():
    c, o, _, _ = plan([2])
    x = torch.full((2, 64), 200.0, device="cuda", dtype=torch.float16)
    w = torch.full((1, 64, 8), 200.0, device="cuda", dtype=torch.float16)
    assert torch.isposinf(X.expert_products(x, w, c, o)).all()


def test_same_result_again_and_on_another_stream():
    c, o, capacity, _ = plan([100, 0, 333, 7], 16)
    x, w, g = matrix(capacity, 264, torch.bfloat16), weights_of(4, 264, 520, torch.bfloat16, "in_out"), None
    g = matrix(capacity, 520, torch.bfloat16, seed=3)
    first = (X.expert_products(x, w, c, o), *X.expert_products_backward(g, x, w, c, o))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = (X.expert_products(x, w, c, o), *X.expert_products_backward(g, x, w, c, o))
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_from_another_host_thread():
    """A thread that has made no CUDA call before."""
    c, o, capacity, _ = plan([100, 30])
    x, w = matrix(capacity, 64, torch.bfloat16), weights_of(2, 64, 72, torch.bfloat16, "in_out")
    here, there = X.expert_products(x, w, c, o), []
    torch.cuda.synchronize()
    thread = threading.Thread(target=lambda: there.append(X.expert_products(x, w, c, o)))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert torch.equal(here, there[0])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [300, 40_000])
def test_segments_on_top_of_each_other_end(rows, dtype):
    """Every expert claims all rows: what does not fit the number of tiles of a plan is left out, the first stays."""
    x, w = matrix(rows, 64, TYPES[dtype]), weights_of(700, 64, 72, TYPES[dtype], "in_out")
    c = torch.full((700,), 1 << 30, dtype=torch.int32, device="cuda")
    o = torch.zeros(701, dtype=torch.int32, device="cuda")
    out = X.expert_products(x, w, c, o)
    assert out.shape == (rows, 72)
    c[1:] = 0
    c[0] = rows
    o[1:] = rows
    out = X.expert_products(x, w, c, o)
    close(out, x.double() @ w[0].double(), x.double().abs() @ w[0].double().abs(), 64)


def test_segments_that_are_no_plan_stay_inside():
    """Counts and offsets beyond the rows are cut there; nothing outside the tensors is touched."""
    x = matrix(40, 64, torch.bfloat16)
    w = weights_of(3, 64, 72, torch.bfloat16, "in_out")
    c = torch.tensor([10, 1 << 30, -5], dtype=torch.int32, device="cuda")
    o = torch.tensor([0, 10, 1 << 30, 2000], dtype=torch.int32, device="cuda")
    out = X.expert_products(x, w, c, o)
    close(out[10:], x[10:].double() @ w[1].double(), x[10:].double().abs() @ w[1].double().abs(), 64)
    grad = X.expert_products_grad_weights(matrix(40, 72, torch.bfloat16, seed=5), x, c, o)
    assert torch.isfinite(grad).all() and not grad[2].any()
