"""Keys and values stored in 8 bits and read back, against the definition in 64 bits: every code and byte has to be the same."""
import numpy as np
import pytest
import torch

from llm_inference_lab_b200.kernels import ops
from q8_helpers import decode, encode, random_pages

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # half a step, relative to the value


def angles(rng, tokens, half):
    a = rng.uniform(0, 30000, (tokens, 1)) * np.power(1e6, -np.arange(half) / max(half, 1))
    return np.stack((np.cos(a), np.sin(a)), axis=-1).astype(np.float32)


def turned(x, table, rotary_dim):
    half = rotary_dim // 2
    c, s = (table[:, None, :, i].astype(np.float64) for i in (0, 1))
    lo, hi = x[..., :half], x[..., half: rotary_dim]
    size = np.abs(lo) + np.abs(hi)
    return (np.concatenate((lo * c - hi * s, hi * c + lo * s, x[..., rotary_dim:]), axis=-1),
            np.concatenate((size, size, np.abs(x[..., rotary_dim:])), axis=-1))


def codes_of(pages):
    return [t.view(torch.uint8).cpu().numpy().copy() for t in pages]


def run_store(rng, tokens, n_q, n_kv, d, rotary_dim, page, dtype, parts=0, rows=None, strided=False, bias=True):
    """Stores rows at shuffled slots, some of them nowhere; checks every byte of the pool and the queries."""
    width = (n_q + 2 * n_kv) * d
    pages = random_pages(ops, rng, -(-tokens // page) + 2, n_kv, page, d)
    before = codes_of(pages)
    if rows is None:
        rows = rng.standard_normal((tokens, width)) * np.exp(2 * rng.standard_normal((tokens, 1)))
    x = torch.from_numpy(rows.astype(np.float32)).cuda()
    b = None
    if parts:
        more = torch.from_numpy(rng.standard_normal((parts - 1, tokens, width)).astype(np.float32)).cuda()
        qkv = torch.cat((x[None], more)).contiguous()
        total = qkv.double().cpu().numpy().sum(axis=0)      # (few numbers of 24 bits: their sum in 64 bits is off by less than 2^-50)
        if bias:
            b = torch.from_numpy(rng.standard_normal(width).astype(np.float32)).cuda().to(torch.bfloat16)
            total = total + b.double().cpu().numpy()
        dtype = torch.bfloat16
        used = torch.from_numpy(total.astype(np.float32)).to(torch.bfloat16).double().numpy()
    else:
        qkv = x.to(dtype)
        if strided:
            wide = torch.zeros((tokens, width + 3), dtype=dtype, device="cuda")
            wide[:, 1: 1 + width] = qkv
            qkv = wide[:, 1: 1 + width]
        used = qkv.double().cpu().numpy()
    table = angles(rng, tokens, rotary_dim // 2)
    slots = rng.permutation(pages.k.shape[0] * page)[:tokens].astype(np.int32)
    if tokens > 2:
        slots[tokens // 2] = -1
    kept = qkv.clone()
    q = ops.rope_kv_store_q8(qkv, torch.from_numpy(table).cuda() if rotary_dim else None, rotary_dim, torch.from_numpy(slots).cuda(), pages,
                             n_q, n_kv, d, bias=b)
    ops.take_device_errors()
    assert torch.equal(qkv, kept) or not np.isfinite(rows).all()
    used = used.reshape(tokens, n_q + 2 * n_kv, d)
    with np.errstate(invalid="ignore"):
        exact, size = turned(used[:, : n_q + n_kv], table, rotary_dim)
    for i, new in ((0, exact[:, n_q:]), (1, used[:, n_q + n_kv:])):
        codes, bytes_ = encode(new)
        for t in np.flatnonzero(slots >= 0):
            before[i][slots[t] // page, :, slots[t] % page] = codes[t]
            before[i + 2][slots[t] // page, :, slots[t] % page] = bytes_[t]
    for name, want, got in zip(("k", "v", "k_scale", "v_scale"), before, codes_of(pages)):
        assert np.array_equal(want, got), f"{name}: {np.mean(want != got):.2g} of the bytes differ"
    if np.isfinite(rows).all():
        # two products and their difference in 32 bits, then one rounding to the type
        off = np.abs(q.double().cpu().numpy().reshape(tokens, n_q, d) - exact[:, :n_q])
        assert (off <= EPS[dtype] * np.abs(exact[:, :n_q]) + 3 * 2.0 ** -24 * size[:, :n_q] * (1 + EPS[dtype])).all()


@pytest.mark.parametrize("tokens", [1, 2, 37, 300])
@pytest.mark.parametrize("n_q, n_kv, d, page", [(14, 2, 64, 16), (28, 4, 128, 16), (3, 3, 256, 8), (2, 1, 16, 5), (4, 2, 32, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store_whole_heads(tokens, n_q, n_kv, d, page, dtype):
    run_store(np.random.default_rng(tokens + d), tokens, n_q, n_kv, d, d, page, dtype)


@pytest.mark.parametrize("n_q, n_kv, d, rotary_dim", [(3, 1, 64, 32), (2, 2, 80, 80), (2, 1, 96, 0), (1, 1, 33, 20), (2, 1, 1, 0), (4, 2, 128, 126)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store_other_sizes(n_q, n_kv, d, rotary_dim, dtype):
    run_store(np.random.default_rng(d), 19, n_q, n_kv, d, rotary_dim, 16, dtype)


@pytest.mark.parametrize("parts", [1, 2, 7, 8, 9, 17])
@pytest.mark.parametrize("tokens, n_q, n_kv, d, rotary_dim", [(8, 14, 2, 64, 64), (3, 4, 2, 128, 128), (2, 2, 1, 256, 256), (5, 2, 1, 48, 48)])
def test_store_sums_parts(parts, tokens, n_q, n_kv, d, rotary_dim):
    run_store(np.random.default_rng(parts), tokens, n_q, n_kv, d, rotary_dim, 16, torch.bfloat16, parts=parts, bias=parts != 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store_rows_off_their_boundaries(dtype):
    run_store(np.random.default_rng(3), 21, 6, 2, 64, 64, 16, dtype, strided=True)


@pytest.mark.parametrize("d, rotary_dim", [(64, 64), (48, 24)])
def test_store_numbers_at_the_borders(d, rotary_dim):
    """Rows of zeros, of one number, of the smallest and the largest, with infinities and NaN; halfway between two codes."""
    rng = np.random.default_rng(0)
    n_q, n_kv = 1, 1
    rows = rng.standard_normal((10, 3 * d))
    rows[0] = 0
    rows[1, d:] = 0
    rows[1, d + 3] = rows[1, 2 * d + 5] = 448.0
    rows[2, d:] *= 1e-39
    rows[3, d:] *= 1e-30
    rows[4, d:] = np.sign(rows[4, d:]) * 1e38
    rows[5, d + 1] = np.inf
    rows[6, 2 * d + 1] = -np.inf
    rows[7, d + 2] = rows[7, 2 * d + 2] = np.nan
    rows[8, 2 * d:] = np.round(rows[8, 2 * d:] * 8) / 8 + 17 / 16          # bfloat16 numbers halfway between codes
    rows[9, 2 * d:] = 0
    rows[9, 2 * d] = -1e-45
    run_store(rng, 10, n_q, n_kv, d, rotary_dim, 16, torch.float32, rows=rows)
    run_store(rng, 10, n_q, n_kv, d, rotary_dim, 16, torch.bfloat16, rows=rows)


@pytest.mark.parametrize("rows", [0, 1, 17, 1000])
@pytest.mark.parametrize("n_kv, d, page", [(2, 64, 16), (4, 128, 16), (1, 33, 7), (3, 20, 8), (2, 4, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_load(rows, n_kv, d, page, dtype):
    rng = np.random.default_rng(rows + d)
    pages = random_pages(ops, rng, 20, n_kv, page, d, spread=8.0)
    pages.k_scale[3] = 255
    slots = rng.integers(-1, 20 * page, rows).astype(np.int32)      # some nowhere, some more than once
    k, v = ops.kv_load_q8(pages, torch.from_numpy(slots).cuda(), dtype)
    ops.take_device_errors()
    for got, codes, scale in ((k, pages.k, pages.k_scale), (v, pages.v, pages.v_scale)):
        want = decode(codes.view(torch.uint8).cpu().numpy(), scale.cpu().numpy()).transpose(0, 2, 1, 3).reshape(-1, n_kv, d)[slots]
        want[slots < 0] = 0
        assert got.dtype == dtype and got.shape == (rows, n_kv, d)
        assert np.array_equal(got.double().cpu().numpy(), want, equal_nan=True)


def test_codes_off_their_boundaries():
    rng = np.random.default_rng(4)
    pages = random_pages(ops, rng, 3, 2, 8, 64)
    moved = []
    for t in pages[:2]:
        raw = torch.empty((t.numel() + 3,), dtype=torch.uint8, device="cuda")
        raw[3:] = t.view(torch.uint8).reshape(-1)
        moved.append(raw[3:].view(torch.float8_e4m3fn).view(t.shape))
    slots = torch.arange(24, dtype=torch.int32, device="cuda")
    for got, want in zip(ops.kv_load_q8(pages._replace(k=moved[0], v=moved[1]), slots), ops.kv_load_q8(pages, slots)):
        assert torch.equal(got, want)


def test_slots_outside_the_pool_are_reported():
    pages = random_pages(ops, np.random.default_rng(0), 3, 2, 16, 64)
    before = codes_of(pages)
    slots = torch.tensor([5, 48, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    ops.kv_load_q8(pages, slots)
    with pytest.raises(ops.KernelError, match="outside the pool"):
        ops.take_device_errors()
    table = torch.ones((1, 32, 2), device="cuda")
    ops.rope_kv_store_q8(torch.ones((1, 6 * 64), dtype=torch.bfloat16, device="cuda"), table, 64, slots[1:2].clone(), pages, 2, 2, 64)
    with pytest.raises(ops.KernelError, match="outside the pool"):
        ops.take_device_errors()
    assert all(np.array_equal(a, b) for a, b in zip(before, codes_of(pages)))


def test_pool_beyond_32_bit_offsets():
    """A pool of more than 2^32 codes: the last page's rows are stored, read back, and attended where they lie."""
    n_kv, page, d, count = 8, 16, 128, (1 << 18) + 3
    pages = ops.quant_pages(count, n_kv, page, d, "cuda")
    assert pages.k.numel() > 1 << 32
    rng = np.random.default_rng(9)
    qkv = torch.from_numpy(rng.standard_normal((5, 24 * d)).astype(np.float32)).cuda().to(torch.bfloat16)
    table = torch.from_numpy(angles(rng, 5, d // 2)).cuda()
    slots = torch.arange(5, dtype=torch.int32, device="cuda") + (count - 1) * page + 2
    q = ops.rope_kv_store_q8(qkv, table, d, slots, pages, 8, n_kv, d)
    small = ops.quant_pages(1, n_kv, page, d, "cuda")
    ops.rope_kv_store_q8(qkv, table, d, slots - (count - 1) * page, small, 8, n_kv, d)
    far, near = ops.kv_load_q8(pages, slots), ops.kv_load_q8(small, slots - (count - 1) * page)
    assert torch.equal(far[0], near[0]) and torch.equal(far[1], near[1])
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    outs = []
    for pool, last in ((pages, count - 1), (small, 0)):
        pool.k_scale[last, :, :2] = pool.v_scale[last, :, :2] = 127
        pool.k[last, :, :2] = pool.v[last, :, :2] = 1.0
        outs.append([ops.attention_q8(x, pool, ints(0, 5), ints(7), ints(2), ints(last)[None], 1, [5], 7, 8, n_kv, d, 0, d ** -0.5)
                     for x in (q, q.float())])
    ops.take_device_errors()
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    del pages, pool
    torch.cuda.empty_cache()
