"""GPU: the 8-bit floating point entries against their formulas in 64 bits.

Tolerances.  A value v on the quantiser's scale is rounded to e4m3: at most half a
step, 2^-4 |v| (normal) or 2^-10 (subnormal).  Before that rounding the f32
arithmetic moves v by a few 2^-24 (product, 448 / g, product; for SwiGLU the
exponential, a sum and a quotient more): SLACK = 2^-20 covers sixteen of them.
Scales take one to five f32 roundings after a sum of k squares, whose own
relative error stays below (k / 256 + 12) 2^-24 (each of 256 or more threads sums
k / 256 terms or fewer, then a tree of 8 levels): 2^-20 up to k = 1024.
A product's sum of 128 exact terms per block, then over the blocks, is off by at
most (128 + blocks + 4) 2^-23 of the sum of magnitudes (2^-23: the tensor cores may
truncate), and the output rounding by eps / 2."""
import pytest
import torch

from agent_harness_b200._lib import AhError, lib

pytestmark = pytest.mark.gpu

G, F, TINY, SLACK = 128, 448.0, 2.0**-100, 2.0**-20
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def fp8(cuda):
    from agent_harness_b200 import fp8 as m
    return m


def randn(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def groups(z):
    """max(|z|, TINY) of each group, and over each column."""
    m, k = z.shape
    p = torch.nn.functional.pad(z.abs(), (0, -k % G)).view(m, -1, G).amax(2).clamp(min=TINY)
    return p, p.repeat_interleave(G, 1)[:, :k]


def check_quantised(q, s, z, row=None, k_sum=1):
    """q, s stand for z * row: z in 64 bits, row the scales' common factor."""
    g, col = groups(z)
    want = g / F * (1.0 if row is None else row)
    tol = SLACK * max(1.0, k_sum / 1024)
    assert ((s.double() - want).abs() <= tol * want).all()
    v = z * F / col
    off = (q.double() - v).abs()
    assert (off <= torch.maximum(v.abs() * 2.0**-4, torch.tensor(2.0**-10, device=v.device).double()) + SLACK * v.abs()).all()


def spread(s, shape):
    return s.double().repeat_interleave(G, 1)[:, : shape[1]] if s.shape[0] == shape[0] else \
        s.double().repeat_interleave(G, 0)[: shape[0]].repeat_interleave(G, 1)[:, : shape[1]]


ROWS = [(1, 1), (1, 128), (1, 4096), (3, 127), (2, 129), (5, 1003), (16, 640), (2, 2048), (33, 264), (300, 160)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", ROWS)
def test_quantize(fp8, m, k, dtype):
    x = randn(m, k, seed=m + k, dtype=dtype)
    q, s = fp8.quantize_fp8(x)
    check_quantised(q, s, x.double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", ROWS)
def test_swiglu(fp8, m, k, dtype):
    gu = randn(m, 2 * k, seed=2 * m + k, dtype=dtype) * 3
    gate, up = gu[:, :k], gu[:, k:]  # strided halves, the second unaligned where k is odd
    q, s = fp8.swiglu_fp8(gate, up)
    g = gate.double()
    check_quantised(q, s, g / (1 + torch.exp(-g)) * up.double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wdtype", TYPES)
@pytest.mark.parametrize("m,k", ROWS)
def test_norm(fp8, m, k, dtype, wdtype):
    x, r = randn(m, k, seed=m * k, dtype=dtype), randn(m, k, seed=m * k + 1, dtype=dtype)
    w = (1 + 0.2 * randn(k, seed=3)).to(wdtype)
    h = (x.float() + r.float()).to(dtype).double()
    q, s = fp8.add_rms_norm_fp8(x, w, residual=r, eps=1e-5)
    assert torch.equal(r.double(), h)
    rs = 1 / (h.square().mean(1, keepdim=True) + 1e-5).sqrt()
    check_quantised(q, s, h * w.double(), rs, k)
    q, s = fp8.add_rms_norm_fp8(x, w, eps=1e-3)
    rs = 1 / (x.double().square().mean(1, keepdim=True) + 1e-3).sqrt()
    check_quantised(q, s, x.double() * w.double(), rs, k)


@pytest.mark.parametrize("k", [16384, 20000, 40001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [3, 400])
def test_long_rows(fp8, m, k, dtype):
    x, w = randn(m, k, seed=k, dtype=dtype), torch.ones(k, device="cuda")
    h = x.double()
    q, s = fp8.add_rms_norm_fp8(x, w)
    check_quantised(q, s, h, 1 / (h.square().mean(1, keepdim=True) + 1e-5).sqrt(), k)
    check_quantised(*fp8.quantize_fp8(x), h)
    r = randn(m, k, seed=k + 1, dtype=dtype)
    h = (x.float() + r.float()).to(dtype).double()
    q, s = fp8.add_rms_norm_fp8(x, w, residual=r)
    assert torch.equal(r.double(), h)
    check_quantised(q, s, h, 1 / (h.square().mean(1, keepdim=True) + 1e-5).sqrt(), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(3, 5), (4, 24), (2, 263), (9, 1030), (301, 517)])
def test_norm_rows_at_every_alignment(fp8, m, k, dtype):
    """Rows of x, residual and w that start at any element of a 16-byte piece, row strides
    odd and even; what lies around the residual's rows stays as it was."""
    for i in range(9):
        for j in (0, 1, 3, 6):
            stride = k + 11 + (i + j) % 3
            xs, rs = randn(m, stride, seed=i, dtype=dtype), randn(m, stride + 1, seed=j + 50, dtype=dtype)
            x, r = xs[:, i:i + k], rs[:, j:j + k]
            w = (1 + 0.2 * randn(k + i, seed=3)).to(dtype)[i // 2:i // 2 + k]
            h = (x.float() + r.float()).to(dtype).double()
            around = rs.clone()
            around[:, j:j + k] = h.to(dtype)
            q, s = fp8.add_rms_norm_fp8(x, w, residual=r)
            assert torch.equal(rs, around)
            rms = 1 / (h.square().mean(1, keepdim=True) + 1e-5).sqrt()
            check_quantised(q, s, h * w.double(), rms, k)
            q, s = fp8.add_rms_norm_fp8(x, w)
            rms = 1 / (x.double().square().mean(1, keepdim=True) + 1e-5).sqrt()
            check_quantised(q, s, x.double() * w.double(), rms, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(2401, 1024), (2403, 1032), (19001, 128), (9502, 264), (4999, 2048)])
def test_many_narrow_rows(fp8, m, k, dtype):
    """Several rows per thread, row counts that leave some of them empty."""
    n = m + 3
    q = torch.full((n, (k + 15) // 16 * 16), 7, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s = torch.full((n, (k + G - 1) // G), -1.0, device="cuda")
    x, u = randn(m, k, seed=m, dtype=dtype), randn(m, k, seed=k, dtype=dtype)
    g = x.double()
    for z in (g, g / (1 + torch.exp(-g)) * u.double()):
        if z is g:
            fp8.quantize_fp8(x, out=q[:m, :k], scales=s[:m])
        else:
            fp8.swiglu_fp8(x, u, out=q[:m, :k], scales=s[:m])
        check_quantised(q[:m, :k], s[:m], z)
        assert (q.view(torch.uint8)[m:] == 7).all() and (s[m:] == -1).all()


def test_many_short_rows(fp8):
    """More rows than a grid's second dimension holds."""
    m, k = 70001, 24
    x = randn(m, k, seed=9, dtype=torch.float16)
    check_quantised(*fp8.quantize_fp8(x), x.double())
    h = x.double()
    q, s = fp8.add_rms_norm_fp8(x, torch.ones(k, device="cuda"))
    check_quantised(q, s, h, 1 / (h.square().mean(1, keepdim=True) + 1e-5).sqrt(), k)


@pytest.mark.parametrize("dtype", TYPES)
def test_zero_and_tiny_rows(fp8, dtype):
    x = torch.zeros(3, 300, dtype=dtype, device="cuda")
    x[1, 5] = 1e-7
    x[2, 130:] = 6.0
    for q, s in (fp8.quantize_fp8(x), fp8.add_rms_norm_fp8(x, torch.ones(300, device="cuda"))):
        assert torch.isfinite(s).all() and (s > 0).all()
        assert (q.float()[x == 0] == 0).all() and (q.float()[x != 0] == F).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_values_stay_in_their_group(fp8, dtype, bad):
    x = randn(4, 700, seed=1, dtype=dtype)
    x[1, 300] = bad
    q, s = fp8.quantize_fp8(x)
    y = q.double() * spread(s, q.shape)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[1, 256:384] = True
    assert torch.equal(y.isnan(), hit)
    one = torch.ones_like(x)
    one[1, 300] = bad
    q, s = fp8.swiglu_fp8(torch.ones_like(x), one)
    assert torch.equal((q.double() * spread(s, q.shape)).isnan(), hit)
    # a norm row's sum carries it: NaN through the row, an infinity leaves zeros elsewhere
    q, s = fp8.add_rms_norm_fp8(x, torch.ones(700, device="cuda"))
    y = q.double() * spread(s, q.shape)
    assert y[1, 256:384].isnan().all() and torch.isfinite(y[[0, 2, 3]]).all()
    rest = torch.cat([y[1, :256], y[1, 384:]])
    assert rest.isnan().all() if bad != bad else (rest == 0).all()


def test_rows_behind_the_last_stay(fp8):
    """Strided outputs: neither the columns past k nor the rows past m are written."""
    m, k = 5, 200
    q = torch.full((m + 2, 224), 7, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s = torch.full((m + 2, 4), -1.0, device="cuda")
    x = randn(m, k, seed=4)
    fp8.quantize_fp8(x, out=q[:m, :k], scales=s[:m, :2])
    check_quantised(q[:m, :k], s[:m, :2], x.double())
    assert (q.view(torch.uint8)[:m, k:] == 7).all() and (q.view(torch.uint8)[m:] == 7).all()
    assert (s[:m, 2:] == -1).all() and (s[m:] == -1).all()


def test_norm_in_place_of_its_input(fp8):
    x = randn(3, 256, seed=5)
    h = 2 * x.double()
    q, s = fp8.add_rms_norm_fp8(x, torch.ones(256, device="cuda"), residual=x)
    assert torch.equal(x.double(), h)
    check_quantised(q, s, h, 1 / (h.square().mean(1, keepdim=True) + 1e-5).sqrt(), 256)


# ---- weights and products --------------------------------------------------------------


def blocks(n, k, seed):
    """A random e4m3 matrix (every finite byte) and block scales over two decades."""
    g = torch.Generator("cuda").manual_seed(seed)
    b = torch.randint(0, 256, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    b[(b & 0x7F) == 0x7F] = 0x3A
    shape = ((n + G - 1) // G, (k + G - 1) // G)
    return b.view(torch.float8_e4m3fn), 10 ** (2 * torch.rand(shape, generator=g, device="cuda") - 4)


def acts(fp8, m, k, seed):
    return fp8.quantize_fp8(randn(m, k, seed=seed) * (1 + 9 * (randn(k, seed=seed + 1) > 2)))


def check_product(y, q, s, wq, ws, k):
    a, w = q.double() * spread(s, q.shape), wq.double() * block_spread(ws, wq.shape)
    want, mag = a @ w.t(), a.abs() @ w.abs().t()
    kb = (k + G - 1) // G
    tol = (G + kb + 4) * 2.0**-23 * mag + want.abs() * torch.finfo(y.dtype).eps / 2 * 1.001
    if y.dtype == torch.float16:
        tol += 2.0**-25
    bad = (y.double() - want).abs() > tol
    assert not bad.any(), (bad.nonzero()[:4].tolist(), int(bad.sum()))


def block_spread(s, shape):
    return s.double().repeat_interleave(G, 0)[: shape[0]].repeat_interleave(G, 1)[:, : shape[1]]


SHAPES = [(1, 128, 128), (1, 1, 1), (1, 4096, 4096), (2, 130, 257), (7, 1003, 1001), (16, 2048, 512), (17, 384, 2000),
          (33, 256, 160), (64, 640, 1280), (65, 129, 127), (127, 1000, 384), (128, 512, 128), (129, 300, 1024),
          (200, 1000, 1000), (256, 1024, 2048), (300, 513, 900), (513, 700, 640), (1030, 900, 1100)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(fp8, m, n, k):
    wq, ws = blocks(n, k, m + n + k)
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    assert W.weight_bytes == n * k + 4 * ws.numel()
    q, s = acts(fp8, m, k, 1)
    for dtype in TYPES:
        check_product(W.matmul(q, s, dtype=dtype), q, s, wq, ws, k)
    W.close()


# tiles of 256 tokens x 256 rows: one token or row past a tile, odd numbers of weight
# tiles, one column block and many, outputs a tensor map can and cannot address
LARGE = [(129, 5000, 130), (300, 4000, 200), (256, 5120, 128), (257, 2433, 1), (513, 2049, 384), (700, 1300, 300),
         (1025, 1152, 520), (2100, 1003, 257), (4100, 640, 96)]


# 33 to 128 tokens: one tile of single CTAs, several tiles each, odd numbers of weight
# tiles, tiles split along K, outputs a tensor map can and cannot address
LARGE += [(33, 25500, 160), (64, 38800, 300), (48, 40960, 1280), (65, 20000, 130), (128, 10240, 384), (127, 40100, 300), (96, 9601, 2048), (100, 4864, 1280), (128, 80000, 96)]
# tiles cut along K over clusters of two, four and eight CTAs, uneven parts
LARGE += [(128, 15000, 1100), (65, 7900, 2100), (127, 5000, 4300), (100, 4864, 4224)]


@pytest.mark.parametrize("m,n,k", LARGE)
def test_matmul_large(fp8, m, n, k):
    wq, ws = blocks(n, k, m + n + k)
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    q, s = acts(fp8, m, k, 1)
    for dtype in TYPES:
        check_product(W.matmul(q, s, dtype=dtype), q, s, wq, ws, k)
    W.close()


# tiles past the last full round of the GPU's pairs, cut along the columns
SPLIT = [(260, 2048, 8192), (300, 1930, 8200), (520, 1200, 6000), (100, 40960, 3200), (2048, 9500, 3200)]
WHOLE = [(512, 1100, 6000), (65, 4300, 16000), (65, 5000, 16000)]  # not split, or inside clusters: no workspace


@pytest.mark.parametrize("m,n,k", SPLIT + WHOLE)
def test_matmul_split_along_the_columns(fp8, m, n, k):
    wq, ws = blocks(n, k, m)
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    need = W.workspace_bytes(m)
    assert (need > 0) == ((m, n, k) in SPLIT)
    q, s = acts(fp8, m, k, 1)
    y = W.matmul(q, s)
    check_product(y, q, s, wq, ws, k)
    if not need:
        return
    check_product(W.matmul(q, s, dtype=torch.bfloat16), q, s, wq, ws, k)
    assert torch.equal(W.matmul(q, s), y)
    # no workspace: no split; one too small: refused, nothing written
    z = torch.full((m, n + 2), -1.0, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    ws_ = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")

    def call(workspace, nbytes):
        return lib().ah_fp8w_matmul(W.handle, q.data_ptr(), q.stride(0), s.data_ptr(), s.stride(0), m, z.data_ptr(),
                                    n + 2, 0, workspace, nbytes, st)

    assert call(ws_.data_ptr(), need - 1) == -1 and call(ws_.data_ptr() + 4, need) == -1
    assert (z == -1).all()
    assert call(None, 0) == 0
    check_product(z[:, :n], q, s, wq, ws, k)
    z.fill_(-1)
    assert call(ws_.data_ptr(), need) == 0  # NaN bit patterns in the workspace
    assert torch.equal(z[:, :n], y) and (z[:, n:] == -1).all()
    W.close()


@pytest.mark.parametrize("m,n_embd,n_ff", [(300, 8192, 1000), (400, 700, 2500), (1500, 256, 1100), (320, 8000, 2000)])
def test_gate_up_weight_as_a_plain_one(fp8, m, n_embd, n_ff):
    """gate | up in one product, whole and split tiles, n_ff not a multiple of 128."""
    (gq, gs), (uq, us), (dq, ds) = ffn_weights(n_embd, n_ff, m)
    block = fp8.Fp8SwigluBlock.from_blocks(gq, gs, uq, us, dq, ds)
    q, s = acts(fp8, m, n_embd, 3)
    for dtype in TYPES:
        gu = block.gate_up.matmul(q, s, dtype=dtype)
        check_product(gu[:, :n_ff], q, s, gq, gs, n_embd)
        check_product(gu[:, n_ff:], q, s, uq, us, n_embd)
    block.close()


@pytest.mark.parametrize("m,n", [(5, 300), (300, 2100), (700, 1500)])
def test_infinite_scales_and_huge_values(fp8, m, n):
    """Scales and sums near the ends of f32 behave as f32 does: an infinite activation
    scale makes its row infinite or NaN, every other row stays finite."""
    k = 512
    wq, ws = blocks(n, k, 2)
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    q, s = acts(fp8, m, k, 3)
    s = s.clone()
    s[2, 1] = float("inf")
    y = W.matmul(q, s)
    rest = torch.ones(m, dtype=torch.bool, device="cuda")
    rest[2] = False
    assert not torch.isfinite(y[2]).any() and torch.isfinite(y[rest]).all()
    s[2, 1] = 1.0
    check_product(W.matmul(q, s), q, s, wq, ws, k)


@pytest.mark.parametrize("m", [1, 3, 40, 260, 900])
def test_matmul_strides_and_rows_behind(fp8, m):
    """Unaligned weight rows, padded activations and scales, an output inside a larger matrix."""
    n, k = (300, 500) if m < 900 else (1500, 500)
    wq, ws = blocks(n, k + 3, 5)
    wq, ws = wq[:, 1:k + 1], ws
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    q0, s0 = acts(fp8, m, k, 2)
    q = torch.full((m + 1, 528), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # NaN past k
    q[:m, :k].copy_(q0)
    s = torch.full((m + 1, 9), float("nan"), device="cuda")
    s[:m, 2:6] = s0
    for off, dtype in ((0, torch.float32), (1, torch.float32), (8, torch.bfloat16), (3, torch.float16)):
        y = torch.full((m + 2, n + 24), -3.0, dtype=dtype, device="cuda")
        out = y[1:m + 1, off:off + n]
        W.matmul(q[:m, :k], s[:m, 2:6], out=out)
        check_product(out, q0, s0, wq, ws, k)
        assert (y[0] == -3).all() and (y[m + 1] == -3).all()
        assert (y[:, :off] == -3).all() and (y[:, off + n:] == -3).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(128, 128), (300, 200), (1, 1000), (513, 640)])
def test_weight_from_float(fp8, n, k, dtype):
    """The stored blocks, seen through a product with one-hot rows."""
    w = randn(n, k, seed=n, dtype=dtype)
    w[:, : min(k, 128)] *= 20
    W = fp8.Fp8Weight.from_float(w)
    j = torch.arange(0, k, 7, device="cuda")
    x = torch.zeros(len(j), k, device="cuda")
    x[torch.arange(len(j), device="cuda"), j] = F
    q, s = fp8.quantize_fp8(x)  # 448 at a scale of 1: exact
    y = W.matmul(q, s).double() / F
    want = w.double().t()[j]
    p = torch.nn.functional.pad(w.double().abs(), (0, -k % G, 0, -n % G))
    g = p.view(p.shape[0] // G, G, -1, G).amax((1, 3)).repeat_interleave(G, 0)[:n].repeat_interleave(G, 1)[:, :k].t()[j]
    half = torch.maximum(want.abs() * 2.0**-4, g / F * 2.0**-10)
    assert ((y - want).abs() <= half + SLACK * (want.abs() + g / F)).all()
    W.close()


@pytest.mark.parametrize("m", [1, 5, 70, 300, 1300])
def test_non_finite_rows_stay_theirs(fp8, m):
    """A NaN in one token's values or scales, or in one weight row, reaches only its outputs."""
    n, k = (400, 384) if m < 300 else (2100, 384)
    wq, ws = blocks(n, k, 8)
    wb = wq.view(torch.uint8).clone()
    wb[270, 200] = 0x7F
    W = fp8.Fp8Weight.from_blocks(wb.view(torch.float8_e4m3fn), ws)
    x = randn(m, k, seed=3)
    if m > 1:
        x[1, 130] = float("nan")
    q, s = fp8.quantize_fp8(x)
    y = W.matmul(q, s)
    want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    want[:, 270] = True
    if m > 1:
        want[1] = True
    assert torch.equal(y.isnan(), want)


def test_empty_batch_and_refusals(fp8):
    wq, ws = blocks(256, 256, 1)
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    q, s = fp8.alloc(0, 256)
    assert W.matmul(q, s).shape == (0, 256)
    q, s = acts(fp8, 4, 256, 1)
    for bad in (lambda: W.matmul(q[:, :128], s[:, :1]), lambda: W.matmul(q, s[:, :1]), lambda: W.matmul(q.float(), s),
                lambda: W.matmul(q, s.half()), lambda: W.matmul(q, s, out=torch.empty(4, 255, device="cuda")),
                lambda: W.matmul(q, s, out=torch.empty(4, 256, dtype=torch.float64, device="cuda")),
                lambda: W.matmul(q, s, out=torch.empty(256, 4, device="cuda").t()),
                lambda: W.matmul(q.view(torch.uint8).clone().view(torch.float8_e4m3fn).cpu(), s),
                lambda: fp8.Fp8Weight.from_blocks(wq, ws[:1]),
                lambda: fp8.quantize_fp8(torch.zeros(4, 8, dtype=torch.float64, device="cuda")),
                lambda: fp8.quantize_fp8(torch.zeros(4, 8, device="cuda").t()),
                lambda: fp8.quantize_fp8(torch.zeros(1, 8, device="cuda").expand(4, 8)),
                lambda: fp8.add_rms_norm_fp8(torch.zeros(4, 8, device="cuda"), torch.ones(7, device="cuda")),
                lambda: fp8.add_rms_norm_fp8(torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda"),
                                             residual=torch.zeros(4, 8, device="cuda", dtype=torch.float16)),
                lambda: fp8.swiglu_fp8(torch.zeros(4, 8, device="cuda"), torch.zeros(4, 9, device="cuda"))):
        with pytest.raises(AhError) as e:
            bad()
        assert e.value.status == -1
    # a q matrix whose rows do not start at multiples of 16 bytes
    odd = torch.empty(4, 257, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :256]
    with pytest.raises(AhError):
        W.matmul(odd, s)


# ---- the block, and the operators together ------------------------------------------------


def ffn_weights(n_embd, n_ff, seed):
    return [blocks(*shape, seed + i) for i, shape in enumerate([(n_ff, n_embd), (n_ff, n_embd), (n_embd, n_ff)])]


FFN = [(1, 256, 384), (1, 1024, 2048), (3, 130, 200), (16, 512, 700), (40, 200, 1000), (130, 384, 512),
       (300, 640, 1030), (600, 256, 300), (320, 8192, 2000), (520, 300, 2200)]
FFN += [(50, 256, 12900), (100, 300, 13000), (128, 256, 19500), (80, 1100, 6500)]  # gate/up tiles of single CTAs


@pytest.mark.parametrize("m,n_embd,n_ff", FFN)
@pytest.mark.parametrize("dtype", TYPES)
def test_ffn_block(fp8, m, n_embd, n_ff, dtype):
    """The block against its own steps, taken one by one and checked in 64 bits.
    The activation's f32 inputs may differ in their last bits between the two, so
    a quantised activation may sit one step (2^-3 |q| or 2^-9) away."""
    (gq, gs), (uq, us), (dq, ds) = ffn_weights(n_embd, n_ff, m)
    gs, us, ds = gs * 0.05, us * 0.05, ds * 0.05
    x, r = randn(m, n_embd, seed=1, dtype=dtype), randn(m, n_embd, seed=2, dtype=dtype)
    w = (1 + 0.1 * randn(n_embd, seed=3)).half()
    block = fp8.Fp8SwigluBlock.from_blocks(gq, gs, uq, us, dq, ds)
    r1, r2 = r.clone(), r.clone()
    y = block(x, w, residual=r1)
    q, s = fp8.add_rms_norm_fp8(x, w, residual=r2)
    assert torch.equal(r1, r2)
    gu = block.gate_up.matmul(q, s)
    check_product(gu[:, :n_ff], q, s, gq, gs, n_embd)
    check_product(gu[:, n_ff:], q, s, uq, us, n_embd)
    a, asc = fp8.swiglu_fp8(gu[:, :n_ff], gu[:, n_ff:])
    step = torch.maximum(a.double().abs() * 2.0**-3, torch.tensor(2.0**-9, device="cuda").double())
    asp, wd = spread(asc, a.shape) if m > 1 else asc.double().repeat_interleave(G, 1)[:, :n_ff], \
        (dq.double() * block_spread(ds, dq.shape))
    want, mag = (a.double() * asp) @ wd.t(), (a.double().abs() * asp) @ wd.abs().t()
    one_step = (step * asp) @ wd.abs().t()
    tol = one_step * 1.01 + (G + (n_ff + G - 1) // G + 4) * 2.0**-22 * mag + want.abs() * torch.finfo(dtype).eps
    if dtype == torch.float16:
        tol += 2.0**-25
    assert ((y.double() - want).abs() <= tol).all()
    # all but a few quantised values agree: the outputs are far nearer than the bound
    assert (y.double() - want).norm() <= (2 * torch.finfo(dtype).eps + 2.0**-7) * want.norm()
    block.close()


def test_ffn_from_float_and_without_residual(fp8):
    m, d, n = 4, 256, 384
    gate, up, down = (randn(*sh, seed=i, dtype=torch.bfloat16) * 0.05 for i, sh in enumerate([(n, d), (n, d), (d, n)]))
    x, w = randn(m, d, seed=9), torch.ones(d, device="cuda")
    block = fp8.Fp8SwigluBlock.from_float(gate, up, down)
    y = block(x, w)
    h = x.double()
    h = h / (h.square().mean(1, keepdim=True) + 1e-5).sqrt()
    g, u = h @ gate.double().t(), h @ up.double().t()
    want = (g / (1 + torch.exp(-g)) * u) @ down.double().t()
    # e4m3 twice per product (2^-4 worst, 2^-5.8 rms each), over 5 roundings in a row
    assert (y.double() - want).norm() <= 5 * 2.0**-4 * want.norm()
    with pytest.raises(AhError):
        block(x[:, :128], w[:128])
    with pytest.raises(AhError):
        fp8.Fp8SwigluBlock.from_float(gate, up[:100], down)


def test_ffn_refuses_before_it_touches_the_residual(fp8):
    d, n = 128, 256
    (gq, gs), (uq, us), (dq, ds) = ffn_weights(d, n, 1)
    block = fp8.Fp8SwigluBlock.from_blocks(gq, gs, uq, us, dq, ds)
    x, r, w = randn(2, d), randn(2, d, seed=1), torch.ones(d, device="cuda")
    before = r.clone()
    y = torch.empty(2, d, device="cuda")
    ws = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    need = block.workspace_bytes(2)

    def call(gu=block.gate_up.handle, dn=block.down.handle, y_p=y.data_ptr(), ldy=d, ydt=0, wsp=ws.data_ptr(), nb=need):
        return lib().ah_fp8_ffn(gu, dn, x.data_ptr(), d, r.data_ptr(), d, 0, w.data_ptr(), 0, 1e-5, 2, y_p, ldy, ydt,
                                wsp, nb, st)

    for bad in (dict(gu=block.down.handle), dict(dn=block.gate_up.handle), dict(y_p=0), dict(ldy=d - 1), dict(ydt=2),
                dict(wsp=0), dict(wsp=ws.data_ptr() + 8), dict(nb=need - 1)):
        assert call(**bad) == -1
    torch.cuda.synchronize()
    assert torch.equal(r, before)
    assert call() == 0


@pytest.mark.parametrize("m", [1, 16, 200])
def test_capture_and_streams(fp8, m):
    """A chain of blocks captured once and replayed on new inputs, and eager calls on two streams at once."""
    d, n = 512, 1024
    blocks_ = [fp8.Fp8SwigluBlock.from_blocks(*[t for p in ffn_weights(d, n, 10 * i) for t in p]) for i in range(3)]
    w = torch.ones(d, device="cuda")
    x, r = randn(m, d, dtype=torch.bfloat16), randn(m, d, seed=1, dtype=torch.bfloat16)

    def chain(x, r):
        y = x
        for b in blocks_:
            y = b(y, w, residual=r)
        return y

    r0 = r.clone()
    want = chain(x, r0)
    torch.cuda.synchronize()
    xs, rs = torch.zeros_like(x), torch.zeros_like(r)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        chain(xs.clone(), rs.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = chain(xs, rs)
    for _ in range(2):
        xs.copy_(x)
        rs.copy_(r)
        graph.replay()
        assert torch.equal(ys, want) and torch.equal(rs, r0)
    outs = []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            ri = r.clone()
            outs.append((chain(x, ri), ri))
    torch.cuda.synchronize()
    for y, ri in outs:
        assert torch.equal(y, want) and torch.equal(ri, r0)
    assert lib().ah_check_device_error(None) == 0


def test_repeats_are_bit_identical(fp8):
    for m, n, k in [(1, 4096, 4096), (16, 1000, 2048), (100, 700, 900), (400, 2500, 1500), (260, 2048, 8192)]:
        wq, ws = blocks(n, k, 3)
        W = fp8.Fp8Weight.from_blocks(wq, ws)
        q, s = acts(fp8, m, k, 4)
        y = W.matmul(q, s)
        for _ in range(5):
            assert torch.equal(W.matmul(q, s), y)


_FRESH = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from agent_harness_b200 import fp8
d, n, m = 512, 1024, int(sys.argv[2])
g = torch.Generator("cuda").manual_seed(1)
block = fp8.Fp8SwigluBlock.from_float(*[torch.randn(*s, generator=g, device="cuda") for s in ((n, d), (n, d), (d, n))])
x, r, w = torch.randn(m, d, generator=g, device="cuda"), torch.zeros(m, d, device="cuda"), torch.ones(d, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = block(x, w, residual=r)
graph.replay()
want = block(x, w, residual=torch.zeros_like(r))
torch.cuda.synchronize()
assert torch.equal(y, want), "captured and eager differ"
"""


@pytest.mark.parametrize("m", [1, 2000])
def test_first_call_may_be_captured(fp8, m):
    """A fresh process whose first products are captured, without an eager call before."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _FRESH, root, str(m)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


_FRESH_PRODUCT = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from agent_harness_b200 import fp8
m = int(sys.argv[2])
W = fp8.Fp8Weight.from_float(torch.randn(8192, 2048, device="cuda"))
q, s = fp8.quantize_fp8(torch.randn(m, 2048, device="cuda"))
y = torch.empty(m, 8192, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    W.matmul(q, s, out=y)
graph.replay()
for _ in range(6):
    assert torch.equal(W.matmul(q, s), y), "captured and eager differ"
"""


@pytest.mark.parametrize("m", [65, 128])
def test_first_clustered_product_may_be_captured(fp8, m):
    """Clusters are counted on the first call, also while that is captured."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _FRESH_PRODUCT, root, str(m)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_operators_on_unlike_streams(fp8):
    """Inputs made on one stream, used on another that waits for it, outputs read on a third."""
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    wq, ws = blocks(700, 512, 4)
    W = fp8.Fp8Weight.from_blocks(wq, ws)
    with torch.cuda.stream(a):
        x = randn(50, 512, seed=6)
        q, s = fp8.quantize_fp8(x)
    b.wait_stream(a)
    with torch.cuda.stream(b):
        y = W.matmul(q, s)
    torch.cuda.current_stream().wait_stream(b)
    for t in (x, q, s, y):
        t.record_stream(torch.cuda.current_stream())
    check_quantised(q, s, x.double())
    check_product(y, q, s, wq, ws, 512)
