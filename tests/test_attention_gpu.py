"""cross_attention, its gradient and prefix_attention on the GPU, each value against the 64-bit oracle and the bound that the
oracle derives for it."""
import itertools
import math

import pytest
import torch

import kermac_b200 as kermac
from kermac_b200 import _native
from oracle import attention_oracle as ao

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(seed, *shape, dtype, by=1.0, layout="nhd"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(*shape, generator=g) * by).to(dtype)
    if layout == "hnd":                                     # heads first in memory
        return x.cuda().transpose(-3, -2).contiguous().transpose(-3, -2)
    if layout == "odd":                                     # rows that start on no 16-byte boundary
        wide = torch.zeros(*shape[:-1], shape[-1] + 3, dtype=dtype, device="cuda")
        wide[..., 1:-2] = x.cuda()
        return wide[..., 1:-2]
    return x.cuda()


def spoil(t, lengths):
    """NaN and infinities behind each length."""
    if lengths is not None and t.shape[0] == len(lengths):
        for l, n in enumerate(lengths):
            n = max(0, min(t.shape[1], n))
            t[l, n::2] = math.nan
            t[l, n + 1::2] = math.inf
    return t


def assert_within(got, want, bound, what):
    got = got.cpu().double()
    assert got.shape == want.shape, what
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, torch.zeros_like(got), (got - want).abs())
    worst = (off / bound.clamp_min(2.0 ** -149)).max() if off.numel() else torch.zeros(())
    worst, holes = float(worst), int(torch.isnan(off).sum())
    assert worst <= 1.0 and holes == 0, f"{what}: {worst:.3g} of the bound, {holes} not a number"


def check_forward(dtype, L, N, M, H, Hk, D, lengths, layout="nhd", scale=None, by=1.0):
    q = make(1, L, N, H, D, dtype=dtype, by=by, layout=layout)
    k, v = (spoil(make(s, L, M, Hk, D, dtype=dtype, layout=layout), lengths) for s in (2, 3))
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = kermac.cross_attention(q, k, v, lengths=lens, scale=scale, return_lse=True)
    want, want_lse, bound, lse_bound = ao.attention(q, k, v, lengths, scale)
    assert_within(out, want, bound, "out")
    assert_within(lse, want_lse, lse_bound, "lse")
    assert _native.device_error_flag() == 0


SHAPES = [          # L, N, M, H, Hk, lengths
    (1, 1, 1, 1, 1, None),
    (2, 1, 700, 4, 4, [700, 333]),
    (3, 2, 129, 8, 1, [0, 129, 64]),
    (2, 17, 40, 6, 2, [39, 1]),
    (1, 130, 257, 2, 2, None),
    (2, 200, 300, 4, 1, [256, 300]),
    (2, 65, 128, 3, 3, [-5, 1000]),
    (1, 300, 1, 2, 1, None),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("D", [64, 128])
def test_forward(dtype, shape, D):
    L, N, M, H, Hk, lengths = shape
    check_forward(dtype, L, N, M, H, Hk, D, lengths)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", [1, 2, 7, 8, 40, 72, 80, 96, 100, 112, 136, 200, 250, 256])
@pytest.mark.parametrize("N", [1, 140])
def test_forward_widths(dtype, D, N):
    check_forward(dtype, 2, N, 150, 4, 2, D, [150, 77])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", ["hnd", "odd"])
@pytest.mark.parametrize("N, D", [(1, 64), (9, 40), (150, 64), (260, 128)])
def test_forward_layouts(dtype, layout, N, D):
    check_forward(dtype, 2, N, 200, 4, 2, D, [200, 131], layout=layout)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N, M", [(1, 20000), (16, 9001), (128, 4000)])
def test_split_keys(dtype, N, M):
    # few blocks and many keys: the keys are divided, some pieces of the shorter entry are empty
    check_forward(dtype, 2, N, M, 2, 1, 64, [M, 40])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M", [511, 512, 800, 1100, 1300, 1600, 1900, 2047, 2100, 2600])
@pytest.mark.parametrize("D, Hk", [(64, 1), (128, 4)])
def test_pieces_of_a_cluster(dtype, M, D, Hk):
    # two to eight pieces of the keys of one token (joined inside the kernel for 16-bit types), and more; an entry without keys
    check_forward(dtype, 3, 1, M, 4, Hk, D, [M, 0, 300])
    q, kp, vp = make(1, 5, 1, 4, D, dtype=dtype), make(2, M, Hk, D, dtype=dtype), make(3, M, Hk, D, dtype=dtype)
    none = torch.zeros(5, 0, Hk, D, dtype=dtype, device="cuda")
    want, _, bound, _ = ao.attention(q, none, none, prefix=(kp, vp))
    assert_within(kermac.prefix_attention(q, kp, vp, none, none), want, bound, "a prefix alone")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N", [1, 256])
@pytest.mark.parametrize("scale, by", [(0.0, 1.0), (3.0, 2.0), (0.125, 30.0)])
def test_scales(dtype, N, scale, by):
    # weights that are all equal, and weights that are almost all zero
    check_forward(dtype, 1, N, 300, 2, 2, 64, None, scale=scale, by=by)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N", [1, 140])
def test_rising_scores(dtype, N):
    # keys in the order of their scores: the running maximum rises with every tile, far beyond any fixed margin
    q = torch.ones(1, N, 1, 64, device="cuda").to(dtype)
    k = (torch.linspace(-40, 40, 1000, device="cuda")[None, :, None, None] / 8).expand(1, 1000, 1, 64).to(dtype).contiguous()
    v = make(3, 1, 1000, 1, 64, dtype=dtype)
    out, lse = kermac.cross_attention(q, k, v, scale=1.0, return_lse=True)
    want, want_lse, bound, lse_bound = ao.attention(q, k, v, scale=1.0)
    assert_within(out, want, bound, "out")
    assert_within(lse, want_lse, lse_bound, "lse")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N", [1, 150])
def test_shared_states_and_shared_queries(dtype, N):
    L, M, H, Hk, D = 3, 170, 4, 2, 64
    q, q1 = make(1, L, N, H, D, dtype=dtype), make(4, N, H, D, dtype=dtype)
    k, v = make(2, M, Hk, D, dtype=dtype), make(3, M, Hk, D, dtype=dtype)
    lengths = torch.tensor([100, 0, 170], dtype=torch.int32, device="cuda")
    want, _, bound, _ = ao.attention(q, k[None], v[None])
    assert_within(kermac.cross_attention(q, k, v), want, bound, "shared states")
    assert_within(kermac.cross_attention(q, k.expand(L, M, Hk, D), v.expand(L, M, Hk, D)), want, bound, "expanded states")
    want, _, bound, _ = ao.attention(q, k[None], v[None], lengths)
    assert_within(kermac.cross_attention(q, k, v, lengths=lengths), want, bound, "shared states, lengths")
    kk, vv = make(5, L, M, Hk, D, dtype=dtype), make(6, L, M, Hk, D, dtype=dtype)
    want, _, bound, _ = ao.attention(q1[None], kk, vv, lengths)
    assert_within(kermac.cross_attention(q1, kk, vv, lengths=lengths), want, bound, "shared queries")


PREFIXES = [        # L, N, M, P, H, Hk, lengths
    (1, 1, 1, 1, 1, 1, None),
    (4, 1, 64, 500, 8, 8, [1, 64, 13, 40]),
    (3, 5, 90, 300, 8, 2, [5, 90, 47]),
    (2, 3, 20, 0, 2, 1, [2, 20]),              # no prefix; one query before the first key
    (2, 3, 20, 40, 2, 1, [0, 1]),              # fewer keys than queries: the prefix alone
    (3, 2, 0, 129, 4, 4, None),                # no own keys
    (40, 1, 30, 700, 4, 2, None),
    (2, 70, 300, 260, 4, 4, [70, 290]),        # a chunk of a prompt
    (2, 1, 9000, 9000, 2, 1, [9000, 3]),
    (1, 2, 0, 0, 2, 1, None),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", PREFIXES, ids=str)
@pytest.mark.parametrize("D", [64, 80, 128])
def test_prefix(dtype, shape, D):
    L, N, M, P, H, Hk, lengths = shape
    q = make(1, L, N, H, D, dtype=dtype)
    k, v = (spoil(make(s, L, M, Hk, D, dtype=dtype), lengths) for s in (2, 3))
    kp, vp = make(4, P, Hk, D, dtype=dtype), make(5, P, Hk, D, dtype=dtype)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = kermac.prefix_attention(q, kp, vp, k, v, lengths=lens, return_lse=True)
    want, want_lse, bound, lse_bound = ao.attention(q, k, v, lengths, prefix=(kp, vp))
    assert_within(out, want, bound, "out")
    assert_within(lse, want_lse, lse_bound, "lse")
    assert _native.device_error_flag() == 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("H, Hk", [(3, 1), (10, 2), (8, 1), (6, 6)])
@pytest.mark.parametrize("D", [64, 80, 128])
def test_heads_of_a_group(dtype, H, Hk, D):
    # groups of 3 and 5 do not divide a tile of 128 rows, groups of 8 and 1 do; an odd number of tiles
    check_forward(dtype, 2, 129, 300, H, Hk, D, [300, 140])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N", [1, 3])
@pytest.mark.parametrize("spread", ["even", "uneven"])
def test_prefix_below_queries_that_lie_apart(dtype, N, spread):
    # queries cut out of a longer tensor: the distance between sequences is not N times that between tokens
    L, M, P, H, Hk, D = 20, 40, 200, 8, 2, 64
    whole = make(1, L, N + (2 if spread == "uneven" else 0), H, D, dtype=dtype)
    q = whole[:, :N]
    k, v = make(2, L, M, Hk, D, dtype=dtype), make(3, L, M, Hk, D, dtype=dtype)
    kp, vp = make(4, P, Hk, D, dtype=dtype), make(5, P, Hk, D, dtype=dtype)
    lengths = torch.tensor([(7 * l) % M + 1 for l in range(L)], dtype=torch.int32, device="cuda")
    want, _, bound, _ = ao.attention(q, k, v, lengths, prefix=(kp, vp))
    assert_within(kermac.prefix_attention(q, kp, vp, k, v, lengths=lengths), want, bound, "out")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N, D", [(1, 64), (1, 128), (40, 64), (40, 128), (40, 200)])
def test_without_scratch(dtype, N, D):
    # a caller that gives no scratch gets the same rows from fewer blocks
    from kermac_b200 import attention
    L, M, H, Hk = 2, 4000 if N == 1 else 1500, 4, 2
    q, k, v = (make(s, L, n, h, D, dtype=dtype) for s, n, h in ((1, N, H), (2, M, Hk), (3, M, Hk)))
    args, _ = attention._marshal(q, k, v, None, None)
    out = torch.empty_like(q)
    args.out = attention._heads(out)
    assert _native.attention_scratch_bytes(args, _native.ATTENTION_CROSS) > 0
    _native.launch_attention(args, _native.ATTENTION_CROSS, torch.cuda.current_stream().cuda_stream)
    want, _, bound, _ = ao.attention(q, k, v)
    assert_within(out, want, bound, "out")
    # with both sets of keys the partial sums are needed, and the gradient needs its sums
    args.prefix, args.k_prefix, args.v_prefix = 10, attention._heads(k[0, :10]), attention._heads(v[0, :10])
    for kind in (_native.ATTENTION_PREFIX, _native.ATTENTION_GRAD):
        args.lse, args.lse_stride_l, args.lse_stride_head = out.data_ptr(), H * N, N
        args.q_batch = args.kv_batch = L
        args.grad_out = args.grad_q = attention._heads(q)
        args.grad_k = args.grad_v = attention._heads(k)
        if kind == _native.ATTENTION_GRAD:
            args.prefix = 0
        with pytest.raises(ValueError, match="scratch"):
            _native.launch_attention(args, kind, torch.cuda.current_stream().cuda_stream)


def test_a_full_device_does_without(monkeypatch):
    from test_grad_split_gpu import full_device
    # the planes of float32 keys take 30 MB
    q, k, v = (make(s, 1, n, 2, 64, dtype=torch.float32) for s, n in ((1, 40), (2, 20000), (3, 20000)))
    want, _, bound, _ = ao.attention(q, k, v)
    out = torch.empty_like(q)
    with full_device():
        kermac.cross_attention(q, k, v, out=out)
    assert_within(out, want, bound, "out")


def test_calls_on_two_streams_at_once():
    dtype, L, N, M, H, D = torch.bfloat16, 2, 1, 3000, 8, 64
    inputs = [[make(10 * i + s, L, n, H, D, dtype=dtype) for s, n in ((1, N), (2, M), (3, M))] for i in range(2)]
    want = [kermac.cross_attention(*x).clone() for x in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for x, stream in zip(inputs, streams):
            with torch.cuda.stream(stream):
                got.append(kermac.cross_attention(*x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def check_grad(dtype, q, k, v, lengths, L, g_by=0.5, layout="nhd", scale=None):
    N, H, D = q.shape[-3:]
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = kermac.cross_attention(q, k, v, lengths=lens, scale=scale, return_lse=True)
    g = make(9, L, N, H, D, dtype=dtype, by=g_by, layout=layout)
    grads = kermac.cross_attention_grad(q, k, v, out, lse, g, lengths=lens, scale=scale)
    four = [t if t.dim() == 4 else t[None] for t in (q, k, v)]
    want = ao.attention_grad(*four, g, lengths, scale)
    for name, got in zip(("grad_q", "grad_k", "grad_v"), grads):
        assert_within(got, *want[name], name)
    assert _native.device_error_flag() == 0


GRAD_SHAPES = SHAPES + [(1, 700, 40, 4, 2, None), (2, 300, 520, 2, 1, [520, 200])]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", GRAD_SHAPES, ids=str)
@pytest.mark.parametrize("D", [64, 128])
def test_grad(dtype, shape, D):
    L, N, M, H, Hk, lengths = shape
    q = make(1, L, N, H, D, dtype=dtype)
    k, v = (spoil(make(s, L, M, Hk, D, dtype=dtype), lengths) for s in (2, 3))
    check_grad(dtype, q, k, v, lengths, L)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", [1, 7, 40, 80, 100, 200, 256])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "odd"])
def test_grad_widths_and_layouts(dtype, D, layout):
    L, N, M, H, Hk, lengths = 2, 70, 150, 4, 2, [150, 77]
    q, k, v = (make(s, L, n, h, D, dtype=dtype, layout=layout) for s, n, h in ((1, N, H), (2, M, Hk), (3, M, Hk)))
    check_grad(dtype, q, spoil(k, lengths), spoil(v, lengths), lengths, L, layout=layout)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N, M", [(20, 140), (150, 300), (140, 100)])      # the last: all keys in one tile
@pytest.mark.parametrize("D", [64, 128])
def test_grad_of_broadcast_inputs(dtype, N, M, D):
    L, H, Hk = 3, 4, 2
    lengths = [M, 0, M // 3]
    q, q1 = make(1, L, N, H, D, dtype=dtype), make(4, N, H, D, dtype=dtype)
    k, v = make(2, L, M, Hk, D, dtype=dtype), make(3, L, M, Hk, D, dtype=dtype)
    k1, v1 = make(5, M, Hk, D, dtype=dtype), make(6, M, Hk, D, dtype=dtype)
    check_grad(dtype, q1, k, v, lengths, L)
    check_grad(dtype, q, k1[None], v1[None], None, L)
    check_grad(dtype, q, k1, v1, lengths, L)
    check_grad(dtype, q1, k1, v1, lengths, L)


@pytest.mark.parametrize("N, M", [(40, 90), (256, 2000)])
@pytest.mark.parametrize("by", [1e-4, 300.0])
def test_float16_gradients_keep_their_range(N, M, by):
    # weights of 1/2000 times gradients of 1e-4 lie below the smallest float16
    q, k, v = (make(s, 1, n, 2, 64, dtype=torch.float16) for s, n in ((1, N), (2, M), (3, M)))
    check_grad(torch.float16, q, k, v, None, 1, g_by=by, scale=0.02)


@pytest.mark.parametrize("N, M, D", [(1, 3000, 64), (300, 2000, 64), (300, 700, 128), (300, 30, 64)])
def test_float32_is_no_less_accurate_than_fp32_products(N, M, D):
    # the bounds above are for the worst case; the errors of products in torch's fp32 are what a caller would get otherwise.
    # Root mean squares over some 10^5 values: a quarter more than theirs is far outside what chance does to them.
    q, k, v, g = (make(s, 1, n, 2, D, dtype=torch.float32, by=by) for s, n, by in ((1, N, 1.5), (2, M, 1.0), (3, M, 1.0), (9, N, 0.5)))
    assert not torch.backends.cuda.matmul.allow_tf32

    def formulas(q, k, v, g):
        q, k, v, g = (t[0].transpose(0, 1) for t in (q, k, v, g))
        s = torch.matmul(q, k.transpose(1, 2)) / math.sqrt(D)
        e = torch.exp(s - s.amax(dim=-1, keepdim=True))
        p = e / e.sum(dim=-1, keepdim=True)
        out = torch.matmul(p, v)
        ds = p * (torch.matmul(g, v.transpose(1, 2)) - (g * out).sum(dim=-1, keepdim=True)) / math.sqrt(D)
        return [t.transpose(0, 1)[None] for t in (out, torch.matmul(ds, k), torch.matmul(ds.transpose(1, 2), q), torch.matmul(p.transpose(1, 2), g))]

    exact, plain = formulas(*(t.double() for t in (q, k, v, g))), formulas(q, k, v, g)
    out, lse = kermac.cross_attention(q, k, v, return_lse=True)
    # The gradient takes its weights from the lse that the caller holds as float32.  That number is off by half a step, 2^-24 of its size,
    # and so is its product with log2(e); lg2.approx adds 2^-22.  An error of lse is a factor on all of a row's weights, which one
    # query does not average away (the formulas above normalise by the sum itself).
    of_lse = 2 * 2.0 ** -24 * float(lse.abs().max()) + 2.0 ** -22
    for i, (got, fp32, want) in enumerate(zip((out, *kermac.cross_attention_grad(q, k, v, out, lse, g)), plain, exact)):
        ours, theirs = ((t.double() - want).square().mean().sqrt() for t in (got, fp32))
        assert ours <= 1.25 * theirs + (2.0 ** -26 if i == 0 else of_lse) * want.square().mean().sqrt(), i


def test_gradient_against_differences():
    # float32, so that a difference of the result has some digits: 1e-2 steps, error of the difference about 1e-4
    L, N, M, H, Hk, D = 1, 6, 9, 2, 1, 8
    q, k, v = (make(s, L, n, h, D, dtype=torch.float32) for s, n, h in ((1, N, H), (2, M, Hk), (3, M, Hk)))
    g = make(9, L, N, H, D, dtype=torch.float32)
    out, lse = kermac.cross_attention(q, k, v, return_lse=True)
    grads = kermac.cross_attention_grad(q, k, v, out, lse, g)

    def loss(*x):
        return float((kermac.cross_attention(*x).double() * g.double()).sum())

    step = 1e-2
    for which, grad in enumerate(grads):
        for at in itertools.islice(range(0, grad.numel(), 7), 12):
            x = [t.clone() for t in (q, k, v)]
            x[which].view(-1)[at] += step
            up = loss(*x)
            x[which].view(-1)[at] -= 2 * step
            difference = (up - loss(*x)) / (2 * step)
            # third derivatives of the softmax times step^2, and 2^-20 of a loss of about 10 over the step
            assert abs(difference - float(grad.view(-1)[at])) < 5e-3


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_equal_calls_give_equal_bits(dtype):
    L, N, M, H, Hk, D = 2, 200, 3000, 4, 2, 64
    q, k, v = (make(s, L, n, h, D, dtype=dtype) for s, n, h in ((1, N, H), (2, M, Hk), (3, M, Hk)))
    g = make(9, L, N, H, D, dtype=dtype)
    first = None
    for _ in range(3):
        out, lse = kermac.cross_attention(q, k, v, return_lse=True)
        now = (out, lse, *kermac.cross_attention_grad(q, k, v, out, lse, g), kermac.prefix_attention(q, k[0], v[0], k, v))
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_destinations_and_rows_that_are_not_there():
    L, N, M, H, Hk, D = 2, 5, 60, 4, 2, 64
    q, k, v = (make(s, L, n, h, D, dtype=torch.bfloat16) for s, n, h in ((1, N, H), (2, M, Hk), (3, M, Hk)))
    lengths = torch.tensor([60, 11], dtype=torch.int32, device="cuda")
    big = torch.full((L, N + 2, H + 1, D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    out = big[:, 1:-1, 1:, 4:-4]                                  # rows on 8-byte boundaries
    lse = torch.full((L, H, N + 3), 7.0, device="cuda")[..., :N]
    got, got_lse = kermac.cross_attention(q, k, v, lengths=lengths, out=out, lse=lse, return_lse=True)
    assert got is out and got_lse is lse
    want, want_lse = kermac.cross_attention(q, k, v, lengths=lengths, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    kept = big.clone()
    kept[:, 1:-1, 1:, 4:-4] = 7.0
    assert torch.all(kept == 7.0)                                 # nothing beside the view was written
    g = make(9, L, N, H, D, dtype=torch.bfloat16)
    plain = kermac.cross_attention_grad(q, k, v, want, want_lse, g, lengths=lengths)
    into = [torch.full((L, n, h + 1, D + 2), 7.0, dtype=torch.bfloat16, device="cuda") for n, h in ((N, H), (M, Hk), (M, Hk))]
    views = [t[:, :, :-1, 1:-1] for t in into]
    given = kermac.cross_attention_grad(q, k, v, out, lse, g, lengths=lengths, grad_q=views[0], grad_k=views[1], grad_v=views[2])
    for a, b, view, whole in zip(plain, given, views, into):
        assert b is view and torch.equal(a, b)
        assert torch.all(whole[:, :, -1] == 7.0) and torch.all(whole[..., 0] == 7.0) and torch.all(whole[..., -1] == 7.0)
    assert torch.all(plain[1][1, 11:] == 0) and torch.all(plain[2][1, 11:] == 0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_empty_extents(dtype):
    def t(*shape):
        return torch.zeros(*shape, dtype=dtype, device="cuda")
    assert kermac.cross_attention(t(0, 3, 2, 8), t(0, 4, 2, 8), t(0, 4, 2, 8)).shape == (0, 3, 2, 8)
    assert kermac.cross_attention(t(2, 0, 2, 8), t(2, 4, 2, 8), t(2, 4, 2, 8)).shape == (2, 0, 2, 8)
    q, k = t(2, 3, 2, 8) + 1, t(2, 0, 2, 8)
    out, lse = kermac.cross_attention(q, k, k, return_lse=True)
    assert torch.all(out == 0) and torch.all(lse == -math.inf)
    grads = kermac.cross_attention_grad(q, k, k, out, lse, q)
    assert torch.all(grads[0] == 0) and grads[1].shape == k.shape and grads[2].shape == k.shape
    none, k = t(2, 0, 2, 8), t(2, 3, 2, 8) + 1
    out, lse = kermac.cross_attention(none, k, k, return_lse=True)
    grads = kermac.cross_attention_grad(none, k, k, out, lse, none)
    assert torch.all(grads[1] == 0) and torch.all(grads[2] == 0) and grads[0].shape == none.shape


@pytest.mark.parametrize("N", [1, 200])
def test_streams_and_graphs(N):
    L, M, H, Hk, D, P = 2, 2000, 4, 2, 64, 600
    q, k, v = (make(s, L, n, h, D, dtype=torch.bfloat16) for s, n, h in ((1, N, H), (2, M, Hk), (3, M, Hk)))
    g, kp, vp = make(9, L, N, H, D, dtype=torch.bfloat16), make(4, P, Hk, D, dtype=torch.bfloat16), make(5, P, Hk, D, dtype=torch.bfloat16)

    def step():
        out, lse = kermac.cross_attention(q, k, v, return_lse=True)
        return (out, lse, *kermac.cross_attention_grad(q, k, v, out, lse, g), kermac.prefix_attention(q, kp, vp, k, v))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # two graphs with workspaces of their own, replayed in turn and at the same time
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step())
        graphs.append(graph)
    for _ in range(3):
        for result in results:
            for t in result:
                t.fill_(math.nan)
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(want, result))
    # new inputs in the captured buffers
    q.mul_(0.5)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(step(), results[0]))


@pytest.mark.parametrize("N", [1, 200])
def test_offsets_beyond_32_bits(N):
    # heads 2^31 elements apart: a cache of 2 * 4.3 GB in which every fourth row of the second head lies behind 2^31
    M, D = 300, 64
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB")
    store = torch.empty((1 << 31) + (1 << 20), dtype=torch.bfloat16, device="cuda")
    small = make(2, 1, M, 2, D, dtype=torch.bfloat16)
    k = store.as_strided((1, M, 2, D), (0, D, 1 << 31, 1))
    k.copy_(small)
    q = make(1, 1, N, 2, D, dtype=torch.bfloat16)
    want, _, bound, _ = ao.attention(q, small, small)
    out, lse = kermac.cross_attention(q, k, k, return_lse=True)
    assert_within(out, want, bound, "out")
    grads = kermac.cross_attention_grad(q, k, k, out, lse, q)
    same = kermac.cross_attention_grad(q, small, small, out, lse, q)
    assert all(torch.equal(a, b) for a, b in zip(grads, same))


def test_a_run_of_them_together():
    """A decoder layer's step as it is used: training against padded states, then tokens written one by one below a shared
    prompt, which must see what one pass over the whole sequence sees."""
    dtype, L, M, H, Hk, D = torch.bfloat16, 3, 90, 8, 2, 64
    lengths = torch.tensor([90, 41, 7], dtype=torch.int32, device="cuda")
    states = make(2, L, M, 2, Hk, D, dtype=dtype)                 # projected keys and values side by side
    k, v = states[:, :, 0], states[:, :, 1]
    q = make(1, L, 20, H, D, dtype=dtype)
    out, lse = kermac.cross_attention(q, k, v, lengths=lengths, return_lse=True)
    grads = kermac.cross_attention_grad(q, k, v, out, lse, out, lengths=lengths)      # of |out|^2 / 2
    found = ao.attention_grad(q, k, v, out, lengths)
    for name, got in zip(("grad_q", "grad_k", "grad_v"), grads):
        assert_within(got, *found[name], name)
    moved = [(t.float() - 0.1 * d.float()).to(dtype) for t, d in zip((q, k, v), grads)]
    want, _, bound, _ = ao.attention(*moved, lengths)
    assert_within(kermac.cross_attention(*moved, lengths=lengths), want, bound, "after a step")

    P, steps = 150, 6
    kp, vp = make(4, P, Hk, D, dtype=dtype), make(5, P, Hk, D, dtype=dtype)
    own_k, own_v = (torch.zeros(L, steps, Hk, D, dtype=dtype, device="cuda") for _ in range(2))
    new_q, new_k, new_v = (make(s, L, steps, h, D, dtype=dtype) for s, h in ((6, H), (7, Hk), (8, Hk)))
    for t in range(steps):
        own_k[:, t], own_v[:, t] = new_k[:, t], new_v[:, t]
        there = torch.full((L,), t + 1, dtype=torch.int32, device="cuda")
        one = kermac.prefix_attention(new_q[:, t:t + 1], kp, vp, own_k, own_v, lengths=there)
        whole_k, whole_v = (torch.cat([a.expand(L, P, Hk, D), b[:, :t + 1]], dim=1) for a, b in ((kp, new_k), (vp, new_v)))
        want, _, bound, _ = ao.attention(new_q[:, t:t + 1], whole_k, whole_v)
        assert_within(one, want, bound, f"token {t}")
    many = kermac.prefix_attention(new_q, kp, vp, new_k, new_v)
    want, _, bound, _ = ao.attention(new_q, new_k, new_v, prefix=(kp, vp))
    assert_within(many, want, bound, "all tokens at once")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N", [1, 100])
def test_same_bits_as_the_ctypes_marshalling(dtype, N, capsys):
    L, M, H, Hk, D, P = 2, 300, 4, 2, 64, 130
    q, g = make(1, L, N, H, D, dtype=dtype), make(9, L, N, H, D, dtype=dtype)
    k, v = make(2, L, M, Hk, D, dtype=dtype), make(3, L, M, Hk, D, dtype=dtype)
    kp, vp = make(4, P, Hk, D, dtype=dtype), make(5, P, Hk, D, dtype=dtype)
    lengths = torch.tensor([300, 120], dtype=torch.int32, device="cuda")
    assert _native.torch_call()
    for options in (dict(), dict(lengths=lengths), dict(lengths=lengths, scale=0.3)):
        out, lse = kermac.cross_attention(q, k, v, return_lse=True, **options)
        slow, slow_lse = kermac.cross_attention(q, k, v, return_lse=True, debug=True, **options)
        assert torch.equal(out, slow) and torch.equal(lse, slow_lse)
        into, into_lse = torch.empty_like(out), torch.empty_like(lse)
        got = kermac.cross_attention(q, k, v, out=into, lse=into_lse, **options)
        assert got is into and torch.equal(into, out) and torch.equal(into_lse, lse)
        for a, b in zip(kermac.cross_attention_grad(q, k, v, out, lse, g, **options),
                        kermac.cross_attention_grad(q, k, v, out, lse, g, debug=True, **options)):
            assert torch.equal(a, b)
        assert torch.equal(kermac.prefix_attention(q, kp, vp, k, v, **options), kermac.prefix_attention(q, kp, vp, k, v, debug=True, **options))
    assert "Launching kernel" in capsys.readouterr().out
    # declined by the extension, refused by the Python layer
    for bad in (dict(k=k.cpu()), dict(scale=-1.0), dict(lengths=lengths.long())):
        with pytest.raises((TypeError, ValueError)):
            kermac.cross_attention(**dict(dict(q=q, k=k, v=v), **bad))


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
@pytest.mark.parametrize("N", [1, 20, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_of_minus_infinity_in_front(dtype, N, D):
    # the first 150 keys have no weight, whatever the level of the others' scores: here at some -40 * 64 / 8, where exp underflows
    q = (torch.rand(1, N, 2, D, generator=torch.Generator().manual_seed(1)) + 0.5).cuda().to(dtype)
    k, v = make(2, 1, 400, 2, D, dtype=dtype), make(3, 1, 400, 2, D, dtype=dtype)
    k -= 5.0
    k[:, :150, :, 0] = -math.inf
    out, lse = kermac.cross_attention(q, k, v, scale=1.0, return_lse=True)
    want, want_lse, bound, lse_bound = ao.attention(q, k[:, 150:], v[:, 150:], scale=1.0)
    assert_within(out, want, bound, "out")
    assert_within(lse, want_lse, lse_bound, "lse")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradient_of_broadcast_inputs_over_an_empty_batch(dtype):
    # a sum over no batch entry is zero, and is written
    def t(*shape):
        return torch.full(shape, 7.0, dtype=dtype, device="cuda")
    lse = torch.zeros(0, 2, 3, device="cuda")
    none = t(0, 3, 2, 8)
    grad_q = t(1, 3, 2, 8)
    kermac.cross_attention_grad(t(1, 3, 2, 8), t(0, 4, 2, 8), t(0, 4, 2, 8), none, lse, none, grad_q=grad_q)
    assert torch.all(grad_q == 0)
    lengths = torch.zeros(0, dtype=torch.int32, device="cuda")
    for M in (0, 4):
        grads = t(1, 3, 2, 8), t(1, M, 2, 8), t(1, M, 2, 8)
        kermac.cross_attention_grad(t(3, 2, 8), t(M, 2, 8), t(M, 2, 8), none, lse, none, lengths=lengths, grad_q=grads[0], grad_k=grads[1],
                                    grad_v=grads[2])
        assert all(torch.all(g == 0) for g in grads)


def grad_rms(dtype, q, k, v, g, grads, lengths=None, exact_delta=False):
    """Root mean squares of the gradients' errors over what rounding alone may cost them, one number each.

    Roundings are independent of one another, so their squares add: at most u |ds| (and u p) of each weight for its product, u of the
    result, and on delta that of the output it is taken from (unless exact_delta), which shifts a whole row of ds by p.  u is the largest
    error of a rounding; its root mean square over the mantissas is sqrt(1 / 3 * 3 / (8 ln 2)) = 0.425 of that, which is the room that this leaves.
    """
    L, N, H, D = g.shape
    M, Hk = k.shape[1:3]
    u, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0
    q, k, v, g = (t.expand(L, *t.shape[1:]).double().transpose(1, 2) for t in (q, k, v, g))
    k, v = (t.repeat_interleave(H // Hk, dim=1) for t in (k, v))
    s = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(D)
    if lengths is not None:
        hidden = torch.arange(M, device="cuda")[None, :] >= torch.tensor(lengths, device="cuda")[:, None]
        s = s.masked_fill(hidden[:, None, None, :], -math.inf)
        k, v = (t.masked_fill(hidden[:, None, :, None], 0.0) for t in (k, v))
    p = torch.softmax(s, dim=-1).nan_to_num(0.0)
    out = torch.matmul(p, v)
    ds = p * (torch.matmul(g, v.transpose(2, 3)) - (g * out).sum(dim=-1, keepdim=True))
    of_delta = (g ** 2 * (u * out.abs() + tiny) ** 2).sum(dim=-1, keepdim=True) * (not exact_delta)
    rows = torch.matmul(p, k) ** 2 * of_delta                       # what a row's error of delta does to grad_q
    keys = torch.matmul((p ** 2 * of_delta).transpose(2, 3), q ** 2)
    found = []
    for name, got, want, off in (("q", grads[0], torch.matmul(ds, k) / math.sqrt(D), (u ** 2 * torch.matmul(ds ** 2, k ** 2) + rows) / D),
                                 ("k", grads[1], torch.matmul(ds.transpose(2, 3), q) / math.sqrt(D),
                                  (u ** 2 * torch.matmul((ds ** 2).transpose(2, 3), q ** 2) + keys) / D),
                                 ("v", grads[2], torch.matmul(p.transpose(2, 3), g), u ** 2 * torch.matmul((p ** 2).transpose(2, 3), g ** 2))):
        if name != "q":
            want, off = (t.unflatten(1, (Hk, H // Hk)).sum(dim=2) for t in (want, off))
        if got.shape[0] == 1:
            want, off = want.sum(dim=0, keepdim=True), off.sum(dim=0, keepdim=True)
        off = off + (u * want.abs() + tiny) ** 2
        found.append(float((got.double().transpose(1, 2) - want).square().mean().sqrt() / off.mean().sqrt()))
    return found


@pytest.mark.parametrize("D", [64, 100, 128])                      # 100: on mma.sync
@pytest.mark.parametrize("v_by, g_by", [(0.01, 1.0), (0.002, 1.0), (1000.0, 1e-3), (1.0, 1e-3), (100.0, 100.0)])
@pytest.mark.parametrize("N, M", [(64, 5000), (300, 600), (200, 100)])
def test_float16_gradients_whatever_the_size_of_the_values(N, M, D, v_by, g_by):
    # the weights' gradients are of the size |dout| |v| / M: far below float16's range, or above it.  q makes up for it in grad_k where the
    # result itself would leave the range.
    q, k, v, g = (make(s, 2, n, h, D, dtype=torch.float16, by=by) for s, n, h, by in ((1, N, 4, 1.0), (2, M, 2, 1.0), (3, M, 2, v_by), (9, N, 4, g_by)))
    lengths = [M, M - M // 3]
    spoil(k, lengths), spoil(v, lengths)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = kermac.cross_attention(q, k, v, lengths=lens, return_lse=True)
    grads = kermac.cross_attention_grad(q, k, v, out, lse, g, lengths=lens)
    found = grad_rms(torch.float16, q, k, v, g, grads, lengths)
    assert all(x <= 1.0 for x in found), found


@pytest.mark.parametrize("D", [128, 136])                          # on the tensor cores and on mma.sync
@pytest.mark.parametrize("M", [2, 200])
def test_float16_gradients_of_values_with_equal_signs(D, M):
    # dout v^T adds up over the channels: 1200 * 2^-10 * 128 = 150 of ds = 75, which once was multiplied by 2^10 and became infinite
    q, k = torch.full((1, 4, 1, D), 0.05, device="cuda").half(), torch.zeros(1, M, 1, D, dtype=torch.float16, device="cuda")
    v = torch.full((1, M, 1, D), 1200.0, device="cuda").half()
    v[:, M // 2:] = -1200.0
    g = torch.full((1, 4, 1, D), 2.0 ** -10, device="cuda").half()
    out, lse = kermac.cross_attention(q, k, v, return_lse=True)
    want = ao.attention_grad(q, k, v, g)
    for name, got in zip(("grad_q", "grad_k", "grad_v"), kermac.cross_attention_grad(q, k, v, out, lse, g)):
        assert_within(got, *want[name], name)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
@pytest.mark.parametrize("D, layout", [(64, "nhd"), (128, "nhd"), (136, "nhd"), (64, "odd")])      # the last two: on mma.sync
@pytest.mark.parametrize("M, keys", [(1030, 2), (1030, 5), (1030, 11), (130, 11), (11, 11)])
def test_sequences_of_few_keys_have_an_exact_delta(dtype, D, layout, M, keys):
    # the accuracy of a sequence does not depend on how far its batch is padded.  From the rounded output this was 0.51 to 0.75.
    H, Hk, N = 8, 4, 300
    q, k, v, g = (make(s, 2, n, h, D, dtype=dtype, by=by, layout=layout)
                  for s, n, h, by in ((1, N, H, 1.5), (2, M, Hk, 1.0), (3, M, Hk, 1.0), (9, N, H, 0.5)))
    lengths = [M, keys]
    spoil(k, lengths), spoil(v, lengths)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = kermac.cross_attention(q, k, v, lengths=lens, return_lse=True)
    grads = kermac.cross_attention_grad(q, k, v, out, lse, g, lengths=lens)
    found = grad_rms(dtype, *(t[1:] for t in (q, k, v, g)), [t[1:] for t in grads], [keys], exact_delta=True)
    # a tenth above 0.425: some 10^5 independent values of grad_q, and 10^3 of the others
    assert found[0] <= 0.47, found
    assert max(found[1:]) <= 0.55, found


@pytest.mark.parametrize("dtype", TYPES[:2], ids=str)             # float16 scores do not get that far
@pytest.mark.parametrize("N, D", [(1, 64), (150, 64), (150, 128), (150, 136)])
def test_a_scale_of_zero_makes_all_weights_equal(dtype, N, D):
    # scores of 2^106 and more, which a factor of 2^-100 in the place of the zero did not make equal
    M = 300
    q = torch.full((1, N, 2, D), 2.0 ** 50, device="cuda").to(dtype)
    k = make(2, 1, M, 2, D, dtype=dtype, by=2.0 ** 50)
    v = make(3, 1, M, 2, D, dtype=dtype)
    out, lse = kermac.cross_attention(q, k, v, scale=0.0, return_lse=True)
    want, want_lse, bound, lse_bound = ao.attention(q * 2.0 ** -50, k * 2.0 ** -50, v, scale=0.0)
    assert_within(out, want, bound, "out")
    assert_within(lse, want_lse, lse_bound, "lse")


@pytest.mark.parametrize("L, N", [(148, 1), (148, 9), (37, 300), (20, 600)])      # as many blocks as there are SMs: the keys are not divided
@pytest.mark.parametrize("D", [64, 128, 136])
def test_float16_weights_below_the_smallest_float16(L, N, D):
    # one key takes nearly all of the weight and has v = 0 (as a first token may); the others' weights of 2^-25 make the result
    M = 20000
    q, k = torch.zeros(L, N, 1, D, dtype=torch.float16, device="cuda"), torch.zeros(1, M, 1, D, dtype=torch.float16, device="cuda")
    q[..., 0], k[:, 7, :, 0] = 4.0, 25.1 * math.log(2.0) / 4
    v = torch.ones_like(k)
    v[:, 7] = 0.0
    k, v = (t.expand(L, M, 1, D).contiguous() for t in (k, v))
    out = kermac.cross_attention(q, k, v, scale=1.0)
    others = (M - 1) * math.exp(-4.0 * float(k[0, 7, 0, 0]))
    # half a step of the result, 2^-11 of it, and of each weight of 2^-25.1 before 2^-33
    assert (out.double() - others / (1.0 + others)).abs().max() <= others * (2.0 ** -11 + 2.0 ** -7) + 2.0 ** -25


def weights_of(q, k, lengths=None, causal_from=None):
    """softmax in the tensors' own arithmetic, (L, H, N, M); key m of the last M - causal_from belongs to query m - causal_from - (length - N)."""
    L, N, H, D = q.shape
    M, Hk = k.shape[1:3]
    s = torch.matmul(q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(H // Hk, dim=1).transpose(2, 3)) / math.sqrt(D)
    at = torch.arange(M, device="cuda")
    if causal_from is not None:
        last = causal_from + (torch.tensor(lengths, device="cuda")[:, None] - N + torch.arange(N, device="cuda")).clamp_min(-1)      # (L, N)
        s = s.masked_fill(at > last[:, None, :, None], -math.inf)
    elif lengths is not None:
        s = s.masked_fill((at >= torch.tensor(lengths, device="cuda")[:, None])[:, None, None, :], -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(dim=-1, keepdim=True)
    return e / total.masked_fill(total == 0.0, 1.0)


ROUNDED = [         # L, N, M, H, Hk, D, lengths, layout: the kernel for few rows, those on tcgen05, those on mma.sync
    (8, 1, 2000, 16, 4, 128, [2000, 500, 1, 0, 1999, 64, 1024, 700], "nhd"),
    (4, 2, 300, 32, 8, 80, None, "hnd"),
    (2, 300, 700, 8, 2, 64, [700, 130], "nhd"),
    (1, 200, 5000, 4, 4, 128, None, "nhd"),
    (2, 100, 333, 6, 2, 40, [333, 200], "hnd"),
    (2, 300, 700, 8, 2, 136, [700, 130], "nhd"),
    (2, 150, 300, 4, 4, 64, None, "odd"),
    (8, 1, 600, 8, 2, 200, None, "nhd"),
]


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
@pytest.mark.parametrize("shape", ROUNDED, ids=str)
def test_16_bit_results_are_as_near_as_their_roundings(dtype, shape):
    # As in grad_rms: half a step of each weight and of the result, squares added; 0.425 of that is what roundings make, and a tenth more is left
    # for chance.  The worst-case bounds above are some ten times that.
    L, N, M, H, Hk, D, lengths, layout = shape
    q, k, v = (make(s, L, n, h, D, dtype=dtype, by=by, layout=layout) for s, n, h, by in ((1, N, H, 1.5), (2, M, Hk, 1.0), (3, M, Hk, 1.0)))
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = kermac.cross_attention(q, k, v, lengths=lens)
    kp, vp, own_k, own_v = k[0, :M // 2].contiguous(), v[0, :M // 2].contiguous(), k[:, M // 2:], v[:, M // 2:]
    below = kermac.prefix_attention(q, kp, vp, own_k, own_v)
    u = torch.finfo(dtype).eps / 2
    q, k, v, kp, vp, own_k, own_v = (t.double() for t in (q, k, v, kp, vp, own_k, own_v))
    whole_k, whole_v = (torch.cat([a.expand(L, *a.shape), b], dim=1) for a, b in ((kp, own_k), (vp, own_v)))
    for what, p, values, result in (("cross", weights_of(q, k, lengths), v, got),
                                    ("prefix", weights_of(q, whole_k, [M - M // 2] * L, causal_from=M // 2), whole_v, below)):
        values = values.transpose(1, 2).repeat_interleave(H // Hk, dim=1)
        want = torch.matmul(p, values)
        off = u ** 2 * torch.matmul(p ** 2, values ** 2) + (u * want.abs()) ** 2
        found = float((result.double().transpose(1, 2) - want).square().mean().sqrt() / off.mean().sqrt())
        assert found <= 0.47, (what, found)


GRADIENTS = [       # L, N, M, H, Hk, D, lengths, layout, broadcast
    (2, 300, 700, 8, 2, 64, [700, 330], "nhd", ""),
    (2, 100, 5000, 4, 2, 128, [5000, 400], "nhd", ""),                   # the keys divided, some pieces of the shorter entry empty
    (3, 40, 4000, 4, 4, 64, [4000, 0, 140], "nhd", "q"),                 # and one q for all
    (4, 700, 300, 4, 2, 128, [300, 150, 0, 299], "hnd", "kv"),           # queries divided
    (4, 700, 300, 4, 2, 80, None, "nhd", "kv"),
    (1, 2000, 200, 8, 1, 96, None, "nhd", ""),
    (2, 300, 700, 8, 2, 136, [700, 330], "nhd", ""),                     # on mma.sync
    (3, 40, 4000, 4, 4, 64, [4000, 0, 140], "odd", "q"),
    (4, 700, 300, 4, 2, 200, [300, 150, 0, 299], "nhd", "kv"),
]


@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
@pytest.mark.parametrize("shape", GRADIENTS, ids=str)
def test_16_bit_gradients_are_as_near_as_their_roundings(dtype, shape):
    L, N, M, H, Hk, D, lengths, layout, broadcast = shape
    q, k, v, g = (make(s, 1 if name in broadcast else L, n, h, D, dtype=dtype, by=by, layout=layout)
                  for s, name, n, h, by in ((1, "q", N, H, 1.5), (2, "k", M, Hk, 1.0), (3, "v", M, Hk, 1.0), (9, "g", N, H, 0.5)))
    if "k" not in broadcast:
        spoil(k, lengths), spoil(v, lengths)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = kermac.cross_attention(q, k, v, lengths=lens, return_lse=True)
    found = grad_rms(dtype, q, k, v, g, kermac.cross_attention_grad(q, k, v, out, lse, g, lengths=lens), lengths)
    # 0.425, and a tenth for chance
    assert max(found) <= 0.47, found


FLOAT32 = [         # L, N, M, H, Hk, D, lengths, layout, broadcast
    (2, 200, 700, 4, 4, 64, [700, 350], "nhd", ""),                      # in three planes
    (2, 200, 700, 8, 2, 64, None, "nhd", ""),
    (3, 100, 500, 6, 2, 40, [500, 33, 129], "hnd", ""),
    (3, 100, 500, 6, 2, 33, None, "odd", ""),
    (3, 100, 500, 4, 4, 64, None, "nhd", "kv"),
    (2, 1, 3000, 8, 2, 64, [3000, 1234], "nhd", ""),                     # on mma.sync
    (2, 200, 700, 8, 2, 128, [700, 350], "nhd", ""),
    (2, 100, 300, 4, 2, 201, None, "odd", ""),
    (2, 100, 30, 4, 2, 64, [30, 11], "nhd", ""),
]


@pytest.mark.parametrize("shape", FLOAT32, ids=str)
def test_float32_forms_are_no_less_accurate_than_fp32_products(shape):
    # test_float32_is_no_less_accurate_than_fp32_products over the forms that it leaves out, and its tolerances.  To the result's is added what the tensor
    # cores cut off, which is of one sign: a chain of two instructions loses up to 2^-23 of the sum at each, half of that in the mean, together
    # 2^-23.  (It shows in single tokens: their fp32 products are summed by another algorithm in torch, with half of the error of larger ones.)
    chopped = 2.0 ** -23
    L, N, M, H, Hk, D, lengths, layout, broadcast = shape
    q, k, v, g = (make(s, 1 if name in broadcast else L, n, h, D, dtype=torch.float32, by=by, layout=layout)
                  for s, name, n, h, by in ((1, "q", N, H, 1.5), (2, "k", M, Hk, 1.0), (3, "v", M, Hk, 1.0), (9, "g", N, H, 0.5)))
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    assert not torch.backends.cuda.matmul.allow_tf32

    def formulas(q, k, v, g):
        kk, vv = (t.expand(L, *t.shape[1:]) for t in (k, v))
        p = weights_of(q, kk, lengths)
        kh, vh = (t.transpose(1, 2).repeat_interleave(H // Hk, dim=1) for t in (kk, vv))
        qh, gh = q.transpose(1, 2), g.transpose(1, 2)
        out = torch.matmul(p, vh)
        ds = p * (torch.matmul(gh, vh.transpose(2, 3)) - (gh * out).sum(dim=-1, keepdim=True)) / math.sqrt(D)
        grads = [torch.matmul(ds, kh)] + [t.unflatten(1, (Hk, H // Hk)).sum(dim=2) for t in (torch.matmul(ds.transpose(2, 3), qh), torch.matmul(p.transpose(2, 3), gh))]
        grads = [grads[0]] + [t.sum(dim=0, keepdim=True) if broadcast else t for t in grads[1:]]
        return [t.transpose(1, 2) for t in (out, *grads)]

    exact, plain = formulas(*(t.double() for t in (q, k, v, g))), formulas(q, k, v, g)
    out, lse = kermac.cross_attention(q, k, v, lengths=lens, return_lse=True)
    of_lse = 2 * 2.0 ** -24 * float(lse[lse != -math.inf].abs().max()) + 2.0 ** -22
    for i, (got, fp32, want) in enumerate(zip((out, *kermac.cross_attention_grad(q, k, v, out, lse, g, lengths=lens)), plain, exact)):
        ours, theirs = ((t.double() - want).square().mean().sqrt() for t in (got, fp32))
        assert ours <= 1.25 * theirs + (chopped if i == 0 else of_lse) * want.square().mean().sqrt(), (i, float(ours / theirs))
    # a prefix and own tokens: both in planes, one of them, neither
    P = M // 3
    kp, vp = k[0, :P].contiguous(), v[0, :P].contiguous()
    own_k, own_v = (t.expand(L, *t.shape[1:])[:, P:].contiguous() for t in (k, v))

    def prefixed(q, kp, vp, own_k, own_v):
        kk, vv = (torch.cat([a.expand(L, *a.shape), b], dim=1) for a, b in ((kp, own_k), (vp, own_v)))
        p = weights_of(q, kk, [M - P] * L, causal_from=P)
        return torch.matmul(p, vv.transpose(1, 2).repeat_interleave(H // Hk, dim=1)).transpose(1, 2)

    want, fp32 = (prefixed(*(t.to(x) for t in (q, kp, vp, own_k, own_v))) for x in (torch.float64, torch.float32))
    ours, theirs = ((t.double() - want).square().mean().sqrt() for t in (kermac.prefix_attention(q, kp, vp, own_k, own_v), fp32))
    assert ours <= 1.25 * theirs + chopped * want.square().mean().sqrt(), float(ours / theirs)


@pytest.mark.parametrize("dtype, size", [(torch.float16, 4096.0), (torch.float16, 5000.0), (torch.float16, 30000.0), (torch.bfloat16, 1.2e6), (torch.bfloat16, 1.0e12),
                                         (torch.float32, 1.2345e6), (torch.float32, 1.0e12)], ids=str)
@pytest.mark.parametrize("N, D", [(1, 64), (150, 64), (1, 128), (150, 128), (1, 136), (150, 136)])
def test_huge_scores_that_are_equal(dtype, size, N, D):
    # the product of a score of 1e9 and more with a scale is rounded by more than float16's exponents hold, of 1e10 by more than float32's
    M = 700
    q, k = torch.full((1, N, 2, D), size, device="cuda").to(dtype), torch.full((1, M, 2, D), size, device="cuda").to(dtype)
    v = make(3, 1, M, 2, D, dtype=dtype)
    got = kermac.cross_attention(q, k, v)
    want, _, bound, _ = ao.attention(q * 0.0, k * 0.0, v)
    assert_within(got, want, bound, "equal weights")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", [64, 136])
def test_captured_gradients_follow_the_lengths(dtype, D):
    # which sequences have few keys is known on the device alone; other inputs, another size of the values and other lengths in the captured buffers
    L, N, M, H, Hk = 3, 70, 700, 4, 2
    q, k, v, g = (make(s, L, n, h, D, dtype=dtype) for s, n, h in ((1, N, H), (2, M, Hk), (3, M, Hk), (9, N, H)))
    lengths = torch.tensor([700, 2, 64], dtype=torch.int32, device="cuda")

    def step():
        out, lse = kermac.cross_attention(q, k, v, lengths=lengths, return_lse=True)
        return (out, lse, *kermac.cross_attention_grad(q, k, v, out, lse, g, lengths=lengths))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for new, by in (([700, 2, 64], 1.0), ([5, 700, 130], 0.01), ([0, 65, 128], 100.0)):
        lengths.copy_(torch.tensor(new, dtype=torch.int32))
        v.copy_(make(13, L, M, Hk, D, dtype=dtype, by=by))
        spoil(v, new)
        for t in captured:
            t.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), captured))
        assert all(torch.isfinite(t).all() for t in captured[2:])
