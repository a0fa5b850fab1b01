"""Linear layers with dense 8-bit weights in scaled blocks on a B200, against 64 bits.

Tolerances: a sum of exact products in fp32 is off by at most a step (2^-23, whatever way it is cut) per addition along its chain: 128 in a
block and one per block; then bias, activation (a slope of at most 1.13, and some 2^-20 of its own) and residual, and half a step of the result's type."""
import pytest
import torch

import void_b200 as void
from void_b200 import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = {0: lambda z: z, 1: lambda z: z.clamp_min(0), 2: lambda z: z / (1 + torch.exp(-1.5957691216 * (z + 0.044715 * z ** 3))), 3: lambda z: z / (1 + torch.exp(-z))}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _dense(t):
    rows, cols = t.values.shape[-2:]
    s = t.scales.double().repeat_interleave(128, -1)[..., :cols]
    if t.block_rows != 1:
        s = s.repeat_interleave(128, -2)[..., :rows, :]
    return t.values.float().double() * s


def _quantised(x, block_rows):
    """Scales and quotients of the definition, in 64 bits."""
    x = x.double().cpu()
    n, k = x.shape
    q, scales = torch.zeros_like(x), torch.zeros((n + block_rows - 1) // block_rows, (k + 127) // 128, dtype=torch.float64)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            part = x[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128]
            scale = 2.0 ** -100
            while scale * 448 < part.abs().max():
                scale *= 2
            scales[i, j] = scale
            v = part / scale
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
            q[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128] = torch.round(v / step) * step
    return q.cuda(), scales.cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("n, k", [(1, 1), (3, 127), (2, 128), (5, 129), (9, 520), (130, 272), (4, 1111)])
def test_quantiser(n, k, block_rows, dtype):
    x = (torch.randn(n, k, generator=_gen(n), device="cuda") * torch.logspace(-3, 3, n, device="cuda")[:, None]).to(dtype)
    x[0, 0] = 448.0
    if n > 1:
        x[1] = 0
        x[n - 1, :128] = 0
        x[n - 1, 0] = torch.finfo(dtype).smallest_normal
    q, scales = _quantised(x, block_rows)
    for given in (x, torch.empty(n, k + 5, dtype=dtype, device="cuda")[:, 2:k + 2].copy_(x), x.t().contiguous().t()):
        got = void.quantize_fp8_blocks(given, block_rows)
        assert got.shape == (n, k) and torch.equal(got.scales.double(), scales) and torch.equal(got.values.float().double(), q)


def test_quantiser_around_448():
    x = torch.zeros(6, 128, device="cuda")
    for i, v in enumerate((448.0, 448.0 * (1 + 2.0 ** -23), 896.0, 0.875, 0.4375, 3.0e38)):
        x[i, 3] = v
    got = void.quantize_fp8_blocks(x, 1)
    assert got.scales.flatten().tolist()[:5] == [1.0, 2.0, 2.0, 2.0 ** -9, 2.0 ** -10]
    assert got.scales[5] == 2.0 ** 120 and got.values.float()[:, 3].tolist()[:5] == [448.0, 224.0, 448.0, 448.0, 448.0]


def test_infinities_and_nan_stay_with_their_token():
    w = void.quantize_fp8_blocks(torch.randn(200, 300, generator=_gen(1), device="cuda"))
    x = torch.randn(70, 300, generator=_gen(2), device="cuda")
    want = void.void_linear(w, x)
    bad = x.clone()
    bad[3, 5], bad[40, 299], bad[69, 130] = float("nan"), float("inf"), -float("inf")
    got = void.void_linear(w, bad)
    broken = torch.tensor([3, 40, 69], device="cuda")
    assert got[broken].isnan().all()
    kept = torch.ones(70, dtype=torch.bool, device="cuda")
    kept[broken] = False
    assert torch.equal(got[kept], want[kept])


def _bound(x, a, z, y, bias, residual, dtype):
    k = x.shape[1]
    size = x.abs() @ a.abs().t()
    err = size * 2.0 ** -23 * (128 + (k + 127) // 128) + (z.abs() + (bias.abs() if bias is not None else 0)) * 2.0 ** -23
    err = 1.13 * err + y.abs() * 2.0 ** -20
    total = y if residual is None else y + residual
    if residual is not None:
        err = err + (y.abs() + residual.abs()) * 2.0 ** -23
    return err + total.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal, total


def _check(got, x, a, bias, act, residual, dtype):
    z = x @ a.t() + (0 if bias is None else bias.double())
    y = ACTS[act](z)
    bound, total = _bound(x, a, z, y, None if bias is None else bias.double(), None if residual is None else residual.double(), dtype)
    assert got.dtype is dtype and got.shape == total.shape
    bad = ~((got.double() - total).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), ((got.double() - total).abs() / bound).max().item(), bad.nonzero()[0].tolist())


def _weights(m, k, seed):
    """A weight with scales that are no powers of two."""
    w = torch.randn(m, k, generator=_gen(seed), device="cuda") * k ** -0.5
    q = void.quantize_fp8_blocks(w)
    return void.FP8BlockTensor(q.values, q.scales * (torch.rand(q.scales.shape, generator=_gen(seed + 1), device="cuda") + 0.5))


SIZES = [(1, 1, 1), (1, 128, 128), (2, 130, 17), (15, 128, 300), (16, 256, 256), (17, 100, 500), (31, 513, 129), (32, 1000, 640), (33, 128, 2048), (64, 300, 1030),
         (65, 260, 128), (100, 129, 777), (128, 128, 1024), (129, 384, 4096), (200, 255, 256), (256, 256, 128), (257, 140, 300), (300, 2500, 3000),
         (512, 130, 200), (513, 1, 129), (700, 4100, 257), (1500, 2001, 300), (2100, 2064, 300), (1111, 640, 640), (3, 20000, 400), (4, 128, 30000)]


@pytest.mark.parametrize("n, m, k", SIZES)
def test_linear(n, m, k):
    w = _weights(m, k, n)
    a = _dense(w)
    for i, dtype in enumerate(TYPES):
        x = torch.randn(n, k, generator=_gen(5), device="cuda").to(dtype)
        xd = _dense(void.quantize_fp8_blocks(x, 1))
        act = (n + i) % 4
        bias = torch.randn(m, generator=_gen(6), device="cuda").to((torch.float32, dtype)[n % 2]) if i != 1 else None
        residual = torch.randn(n, m, generator=_gen(7), device="cuda").to((dtype, torch.float32)[i % 2]) if i != 2 else None
        got = void.void_linear(w, x, bias, act, residual=residual)
        _check(got, xd, a, bias, act, residual, dtype)
        given = void.void_linear(w, void.quantize_fp8_blocks(x, 1), bias, act, residual=residual, out_dtype=dtype)
        assert torch.equal(given, got)
    assert void.void_linear(w, void.quantize_fp8_blocks(x, 1)).dtype is torch.float32
    void.check_device_status()


def test_the_same_every_time_and_in_any_batch():
    """A token's result depends on the token alone where the launch cuts k the same way, and on nothing from run to run."""
    w = _weights(700, 1500, 1)
    x = torch.randn(600, 1500, generator=_gen(2), device="cuda")
    want = void.void_linear(w, x)
    for _ in range(3):
        assert torch.equal(void.void_linear(w, x), want)


def test_scales_with_strides_of_their_own():
    w = _weights(300, 520, 3)
    x = void.quantize_fp8_blocks(torch.randn(50, 520, generator=_gen(4), device="cuda"), 1)
    want = void.void_linear(w, x)
    scales = torch.full((7, 9), float("nan"), device="cuda")
    scales[1:6, 2:5] = w.scales.t()
    xs = torch.full((50, 12), float("nan"), device="cuda")
    xs[:, ::2][:, :5] = x.scales
    again = void.void_linear(void.FP8BlockTensor(w.values, scales[1:6, 2:5].t()), void.FP8BlockTensor(x.values, xs[:, ::2][:, :5]))
    assert torch.equal(again, want)
    loose = void.FP8BlockTensor(torch.empty(300, 521, dtype=torch.uint8, device="cuda")[:, 1:].copy_(w.values.view(torch.uint8)).view(torch.float8_e4m3fn), w.scales)
    assert torch.equal(void.void_linear(loose, x), want)


def test_weights_are_read_at_the_call():
    w = _weights(256, 256, 5)
    x = torch.randn(20, 256, generator=_gen(6), device="cuda")
    first = void.void_linear(w, x)
    w.scales.mul_(2)
    assert torch.equal(void.void_linear(w, x), first * 2)
    w.values.copy_(torch.zeros_like(w.values))
    assert (void.void_linear(w, x) == 0).all()


def test_weights_scales_and_biases_written_just_before():
    """The product reads its weights ahead of the end of the kernel that quantises x: nothing else may still be under way then."""
    n, m, k = 24, 4096, 4096
    given = [_weights(m, k, s) for s in (1, 2)]
    biases = [torch.randn(m, generator=_gen(s), device="cuda") for s in (3, 4)]
    x = torch.randn(n, k, generator=_gen(5), device="cuda")
    want = [void.void_linear(w, x, b) for w, b in zip(given, biases)]
    w, bias = void.FP8BlockTensor(given[0].values.clone(), given[0].scales.clone()), biases[0].clone()
    got = []
    for i in range(40):
        bias.copy_(biases[i % 2])
        w.scales.copy_(given[i % 2].scales)
        w.values.view(torch.uint8).copy_(given[i % 2].values.view(torch.uint8))
        got.append(void.void_linear(w, x, bias))
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2]), i
    # and what the operator itself brings into place: a residual that is copied, biases of another type, a plan of many experts
    E = 40
    experts = void.quantize_fp8_blocks(torch.randn(E, 128, 256, generator=_gen(6), device="cuda"))
    tokens = torch.randn(400, 256, generator=_gen(7), device="cuda")
    offsets = torch.arange(E + 1, device="cuda") * 10
    want = void.void_expert_linear(experts, tokens, offsets)
    for _ in range(20):
        offsets.zero_()
        offsets.add_(torch.arange(E + 1, device="cuda") * 10)
        assert torch.equal(void.void_expert_linear(experts, tokens, offsets), want)
    r = torch.randn(m, n, generator=_gen(8), device="cuda").double()
    want = void.void_linear(w, x, bias.float(), residual=r.t().float().contiguous())
    for _ in range(20):
        assert torch.equal(void.void_linear(w, x, bias.double(), residual=r.float().t()), want)


def test_results_that_are_given():
    w = _weights(300, 256, 7)
    x = torch.randn(40, 256, generator=_gen(8), device="cuda").half()
    r = torch.randn(40, 300, generator=_gen(9), device="cuda").half()
    want = void.void_linear(w, x, residual=r)
    outer = torch.full((40, 333), 7.0, dtype=torch.float16, device="cuda")
    out = outer[:, 11:311]
    version = out._version
    assert void.void_linear(w, x, residual=r, out=out) is out and out._version > version
    assert torch.equal(out, want) and (outer[:, :11] == 7).all() and (outer[:, 311:] == 7).all()
    stream = r.clone()
    assert torch.equal(void.void_linear(w, x, residual=stream, out=stream), want)
    both = torch.zeros(41 * 300, dtype=torch.float16, device="cuda")
    both[:12000] = r.flatten()
    assert torch.equal(void.void_linear(w, x, residual=both[:12000].view(40, 300), out=both[300:].view(40, 300)), want)
    square = _weights(256, 256, 3)
    want = void.void_linear(square, x)
    assert torch.equal(void.void_linear(square, x, out=x), want)              # (x is read before)
    with pytest.raises(_lib.VoidB200Error, match="out must be"):
        void.void_linear(w, x, out=torch.empty(40, 300, device="cuda"), out_dtype=torch.float16)
    with pytest.raises(_lib.VoidB200Error, match="out must be"):
        void.void_linear(w, x, out=torch.empty(40, 299, dtype=torch.float16, device="cuda"))
    with pytest.raises(_lib.VoidB200Error, match="weights"):
        room = torch.zeros(40 * 300, device="cuda")
        void.void_linear(void.FP8BlockTensor(w.values, room[100:106].view(3, 2)), x, out=room.view(40, 300))
    assert void.void_linear(w, x[:0]).shape == (0, 300)


def test_refusals():
    w = _weights(256, 256, 1)
    e = void.FP8BlockTensor(w.values.view(2, 128, 256), w.scales.view(2, 1, 2))
    x, tokens = torch.randn(256, 256, device="cuda"), void.quantize_fp8_blocks(torch.randn(256, 256, device="cuda"), 1)
    offsets = torch.tensor([0, 100, 256], device="cuda")
    for call, text in [
            (lambda: void.void_linear(tokens, x), "128 x 128"), (lambda: void.void_linear(w, w), "each token"), (lambda: void.void_linear(w, x.double()), "float32"),
            (lambda: void.void_linear(w, x, out_dtype=torch.float64), "output dtype"), (lambda: void.void_linear(w, x, activation=7), "activation code"),
            (lambda: void.void_expert_linear(e, w, offsets), "each token"), (lambda: void.void_expert_linear(e, x.int(), offsets), "float32"),
            (lambda: void.void_linear(void.FP8BlockTensor(w.values.cpu(), w.scales.cpu()), x), "no CPU path"),
            (lambda: void.void_linear(w, x.cpu()), "no CPU path"), (lambda: void.void_linear(w, x, residual=x.cpu()), "GPU only")]:
        with pytest.raises(_lib.VoidB200Error, match=text):
            call()


EXPERTS = [  # runs, rows behind them, M, K
    ([1], 0, 128, 128), ([0, 0, 3], 0, 130, 200), ([5, 0, 40, 1], 7, 300, 257), ([100, 30, 0, 200], 0, 256, 512), ([300, 260, 1, 0, 15], 13, 140, 300),
    ([0, 0], 20, 128, 256), ([700, 2, 600], 1, 260, 640), ([900, 0, 333], 40, 2001, 200), ([17] * 40, 3, 64, 128), ([1] * 70, 0, 200, 384), ([0] * 5 + [513], 0, 129, 129)]


@pytest.mark.parametrize("runs, spare, m, k", EXPERTS)
def test_experts(runs, spare, m, k):
    E, n = len(runs), sum(runs) + spare
    w = _weights(m * E, k, 2) if m % 128 == 0 else None
    if w is None:
        parts = [_weights(m, k, e) for e in range(E)]
        values = torch.stack([p.values.view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn)
        w = void.FP8BlockTensor(values, torch.stack([p.scales for p in parts]))
    else:
        w = void.FP8BlockTensor(w.values.reshape(E, m, k), w.scales.reshape(E, m // 128, -1))
    a = _dense(w)
    ends = torch.tensor([0] + runs).cumsum(0)
    for i, dtype in enumerate(TYPES):
        x = torch.randn(n, k, generator=_gen(5), device="cuda").to(dtype)
        x[sum(runs):] = float("nan")
        xd = _dense(void.quantize_fp8_blocks(x, 1))
        bias = torch.randn(E, m, generator=_gen(6), device="cuda").to(dtype) if i != 2 else None
        act = (E + i) % 4
        got = void.void_expert_linear(w, x, ends.to((torch.int32, torch.int64)[i % 2]).cuda(), bias, act)
        for e in range(E):
            if runs[e]:
                _check(got[ends[e]:ends[e + 1]], xd[ends[e]:ends[e + 1]], a[e], None if bias is None else bias[e], act, None, dtype)
        assert (got[sum(runs):] == 0).all()
        out = torch.full((n, m), 5.0, dtype=dtype, device="cuda")
        void.void_expert_linear(w, void.quantize_fp8_blocks(x, 1) if n else x, ends.cuda(), bias, act, out=out)
        assert torch.equal(out[:sum(runs)], got[:sum(runs)]) and (out[sum(runs):] == 5).all()
    void.check_device_status()


def test_offsets_are_not_trusted():
    w = void.quantize_fp8_blocks(torch.randn(3, 128, 128, generator=_gen(1), device="cuda"))
    x = torch.randn(50, 128, generator=_gen(2), device="cuda")
    for bad in ([5, 20, 10, 50], [0, 10, 20, 51], [-3, 10, 20, 50], [0, 2 ** 40, 20, 50]):
        void.void_expert_linear(w, x, torch.tensor(bad, device="cuda"))
        with pytest.raises(_lib.VoidB200Error, match="offsets"):
            void.check_device_status()
    y = void.void_expert_linear(w, x, torch.tensor([5, 20, 20, 40], device="cuda"))
    assert (y[:5] == 0).all() and (y[40:] == 0).all()
    want = void.void_linear(void.FP8BlockTensor(w.values[0], w.scales[0]), x)
    assert torch.equal(y[5:20], want[5:20])
    void.check_device_status()


def test_expert_refusals():
    w = void.quantize_fp8_blocks(torch.randn(3, 128, 128, generator=_gen(1), device="cuda"))
    x, offsets = torch.randn(50, 128, device="cuda"), torch.tensor([0, 10, 20, 50], device="cuda")
    with pytest.raises(_lib.VoidB200Error, match="vector of 4"):
        void.void_expert_linear(w, x, offsets[:3])
    with pytest.raises(_lib.VoidB200Error, match="int32 or int64"):
        void.void_expert_linear(w, x, offsets.float())
    with pytest.raises(_lib.VoidB200Error, match="activation code"):
        void.void_expert_linear(w, x, offsets, activation=4)
    with pytest.raises(_lib.VoidB200Error, match="out must be"):
        void.void_expert_linear(w, x, offsets, out=torch.empty(49, 128, device="cuda"))


def test_a_wait_that_runs_out_is_reported():
    """The first stage of the ring is never filled: the kernel gives up after a tenth of a second and says so, and the next product is right."""
    import ctypes
    w, x = _weights(300, 700, 1), void.quantize_fp8_blocks(torch.randn(40, 700, generator=_gen(2), device="cuda"), 1)
    want = void.void_linear(w, x)
    out = torch.empty_like(want)
    status = _lib.status_word(x.device)
    a = _lib.Fp8Args(a=w.values.data_ptr(), lda=w.values.stride(0), a_scale=w.scales.data_ptr(), a_scale_row=w.scales.stride(0), a_scale_col=1,
                     x=x.values.data_ptr(), ldx=x.values.stride(0), x_scale=x.scales.data_ptr(), x_scale_row=x.scales.stride(0),
                     x_scale_col=x.scales.stride(1), out=out.data_ptr(), ldc=300, M=300, K=700, N=40, test_hooks=100 | 1 << 16, status=status.data_ptr())
    assert _lib.load().void_fp8_linear(ctypes.byref(a), None, _lib.stream_ptr(x.device)) == 0
    with pytest.raises(_lib.VoidB200Error, match="wait gave up"):
        void.check_device_status()
    assert torch.equal(void.void_linear(w, x), want)
    void.check_device_status()


def test_captured_products_of_two_graphs():
    w = _weights(500, 640, 1)
    experts = void.quantize_fp8_blocks(torch.randn(4, 200, 500, generator=_gen(2), device="cuda"))
    x, offsets = torch.randn(90, 640, generator=_gen(3), device="cuda"), torch.tensor([0, 20, 20, 60, 90], device="cuda")

    def both():
        return void.void_expert_linear(experts, void.void_linear(w, x, None, 3), offsets)
    both()
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(both())
        graphs.append(g)
    for k in range(3):
        x.copy_(torch.randn(90, 640, generator=_gen(10 + k), device="cuda"))
        offsets.copy_(torch.tensor([[0, 1, 50, 50, 90], [10, 20, 30, 40, 50], [0, 0, 0, 0, 0]][k]))
        for g in graphs:
            g.replay()
        want = both()
        assert torch.equal(results[0], want) and torch.equal(results[1], want)


def test_a_capture_without_a_call_before():
    w, x = _weights(1536, 1300, 1), torch.randn(11, 1300, generator=_gen(2), device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = void.void_linear(w, x)
    g.replay()
    assert torch.equal(y, void.void_linear(w, x))


def test_streams():
    w = _weights(1000, 2000, 1)
    x = torch.randn(40, 2000, generator=_gen(2), device="cuda")
    want = void.void_linear(w, x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(void.void_linear(w, x))
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in got)


def test_a_served_layer_of_experts():
    """Router, dispatch, two layers of 8-bit experts and the way back to the residual stream, each against 64 bits on what the one before gave (a
    value next to a border of e4m3 may be rounded either way)."""
    n, d, h, E, top = 37, 256, 384, 8, 2
    up, down = (void.quantize_fp8_blocks(torch.randn(E, *s, generator=_gen(4), device="cuda") * 0.06) for s in ((h, d), (d, h)))
    x, gate = torch.randn(n, d, generator=_gen(5), device="cuda").bfloat16(), torch.randn(d, E, generator=_gen(6), device="cuda").bfloat16()
    ids, weights = void.void_route(x @ gate, top)
    rows, routes = void.void_dispatch(x, ids, E)
    hidden = void.void_expert_linear(up, rows, routes.offsets, None, 3)
    back = void.void_expert_linear(down, hidden, routes.offsets)
    y = void.void_combine(back, routes, weights, residual=x)
    a, b = _dense(up), _dense(down)
    tokens, inner = _dense(void.quantize_fp8_blocks(x, 1)), _dense(void.quantize_fp8_blocks(hidden, 1))
    want, size = x.double(), x.double().abs()
    for t in range(n):
        for j in range(top):
            e, row = int(ids[t, j]), int(routes.position[t, j])
            _check(hidden[row][None], tokens[t][None], a[e], None, 3, None, torch.bfloat16)
            _check(back[row][None], inner[row][None], b[e], None, 0, None, torch.bfloat16)
            part = weights[t, j].double() * back[row].double()
            want[t] += part
            size[t] += part.abs()
    assert ((y.double() - want).abs() <= size * 2.0 ** -24 * 4 + want.abs() * 2.0 ** -8).all()
