"""Attention over latent vectors on the device (llmp_hip_rope, llmp_hip_latent_*) against its operators' definitions in 64 bits
(tests/latent_plain.py), within what their stated roundings give."""
import math

import pytest
import torch

import latent_plain as plain
from llmp_amd import ops

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def normal(g, *shape, dtype=torch.float32, size=1.0):
    return (torch.randn(shape, generator=g) * size).to(dtype)


def within(got, want, bound, name=""):
    over = (got.double().cpu() - want).abs() / bound
    over = torch.where(got.double().cpu() == want, 0.0, over.nan_to_num(nan=math.inf))
    assert over.numel() == 0 or over.max() <= 1.0, f"{name}: {float(over.max()):.3g} of the bound at {torch.nonzero(over == over.max())[0].tolist()}"


# ---------------------------------------------------------------- rotations


def rotation_bound(want, x, dtype):
    """cosine and sine off by 2^-23 (their sums' terms, the phase's 2^-32 turns and a factor's F32), products and their sum
    three roundings of 2^-24, the result's own; all of the pair's size."""
    size = x.abs().amax(-1, keepdim=True) * 2.0
    return size * (2.0 ** -22 + 3 * 2.0 ** -24) + want.abs() * plain.HALF[dtype] * 1.01 + plain.LEAST[dtype]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,head_dim,first,n_dims", [(1, 1, 2, 0, 2), (3, 5, 192, 128, 64), (65, 2, 80, 48, 32), (7, 3, 50, 10, 28), (1100, 1, 64, 0, 64),
                                                               (2, 3, 1040, 8, 1024), (33, 128, 64, 0, 64), (300, 9, 128, 0, 64)])
def test_rope(device, dtype, layout, tokens, heads, head_dim, first, n_dims):
    g = torch.Generator().manual_seed(tokens + head_dim)
    x = normal(g, tokens, heads, head_dim, dtype=TYPES[dtype])
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g, dtype=torch.int32)
    positions[0] = 0
    options = [dict(), dict(freq_scale=1 / 40, ext_factor=1.0, corr_dims=(3.0, 11.0)),
               dict(freq_scale=0.25, freq_factors=(1.0 + torch.rand(n_dims // 2, generator=g) * 7.0).tolist())][tokens % 3]
    table = ops.rope_table(n_dims, 10000.0, **options)
    freqs = plain.frequencies(n_dims, 10000.0, **options)
    size = 1.0 + 0.1 * math.log(40.0) if options.get("ext_factor") else 1.0
    assert table["magnitude"] == pytest.approx(size)
    part = x[..., first:first + n_dims]
    for inverse in (False, True):
        want = plain.rotate(part, positions, freqs, layout, size, inverse)
        got = ops.rope(x.to(device), positions.to(device), table, layout=layout, first=first, inverse=inverse).cpu()
        assert torch.equal(got[..., :first], x[..., :first]) and torch.equal(got[..., first + n_dims:], x[..., first + n_dims:])
        within(got[..., first:first + n_dims], want, rotation_bound(want, part.double(), TYPES[dtype]), f"inverse {inverse}")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_strides_in_place_and_views(device, layout):
    """A view of part of every head, in place; the rest of the memory keeps its values; strides no multiple of 16 bytes."""
    g = torch.Generator().manual_seed(5)
    table = ops.rope_table(64, 500000.0)
    freqs = plain.frequencies(64, 500000.0)
    positions = torch.tensor([0, 5, 131071, 1 << 30], dtype=torch.int32)
    for extra in (0, 1):
        whole = normal(g, 4, 6, 200 + extra, dtype=torch.bfloat16).to(device)
        before = whole.cpu()
        x = whole[:, 1:5, 128:192]
        out = ops.rope(x, positions.to(device), table, layout=layout, out=x)
        assert out is x
        want = plain.rotate(before[:, 1:5, 128:192], positions, freqs, layout)
        within(whole[:, 1:5, 128:192], want, rotation_bound(want, before[:, 1:5, 128:192].double(), torch.bfloat16))
        after = whole.cpu()
        after[:, 1:5, 128:192] = before[:, 1:5, 128:192]
        assert torch.equal(after, before)
        other = torch.zeros(4, 4, 96, dtype=torch.bfloat16, device=device)[..., 16:80]
        ops.rope(whole[:, 1:5, 128:192], positions.to(device), table, layout=layout, inverse=True, out=other)
        within(other, before[:, 1:5, 128:192].double(), 2 * rotation_bound(before[:, 1:5, 128:192].double(), before[:, 1:5, 128:192].double(), torch.bfloat16) +
               before[:, 1:5, 128:192].abs().amax(-1, keepdim=True).double() * 2.0 ** -7)  # there and back: the rounding between them


def test_rope_positions_far_and_negative(device):
    """Phases are exact at any 32-bit position, and the inverse undoes the rotation."""
    positions = torch.tensor([-1, -(1 << 31), (1 << 31) - 1, 123456789, -987654321], dtype=torch.int32)
    x = torch.randn(5, 3, 64)
    table, freqs = ops.rope_table(64, 10000.0), plain.frequencies(64, 10000.0)
    got = ops.rope(x.to(device), positions.to(device), table)
    # Angles in 64 bits, off by 2^-53 of 2^31 at most: 2^-22.
    want = plain.rotate(x, positions, freqs, "half")
    within(got, want, rotation_bound(want, x.double(), torch.float32) + 2.0 ** -20)
    back = ops.rope(got, positions.to(device), table, inverse=True)
    within(back, x.double(), 2 * rotation_bound(x.double(), x.double(), torch.float32))


def test_rope_gradient_is_the_inverse(device):
    """y = R x: the gradient of y . w is R^T w, by the formula and by differences."""
    g = torch.Generator().manual_seed(3)
    x, w = normal(g, 9, 2, 64), normal(g, 9, 2, 64)
    positions = torch.arange(9, dtype=torch.int32) * 1000
    table, freqs = ops.rope_table(64), plain.frequencies(64, 10000.0)
    grad = ops.rope(w.to(device), positions.to(device), table, layout="interleaved", inverse=True).double().cpu()
    leaf = x.double().requires_grad_()
    (plain.rotate(leaf, positions, freqs, "interleaved") * w.double()).sum().backward()
    within(grad, leaf.grad, rotation_bound(leaf.grad, w.double(), torch.float32))
    # The rotation is linear: a difference over one channel is its column.
    step = torch.zeros_like(x)
    step[:, :, 7] = 1.0
    column = ops.rope((x + step).to(device), positions.to(device), table, layout="interleaved").double() - ops.rope(x.to(device), positions.to(device), table, layout="interleaved").double()
    slope = (column.cpu() * w.double()).sum(-1)
    assert (slope - grad[:, :, 7]).abs().max() < 64 * 2.0 ** -20


# ---------------------------------------------------------------- store and read


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kept,width,rope,page", [("bf16", 512, 64, 16), ("f16", 256, 32, 48), ("bf16", 256, 64, 256), ("f16", 512, 32, 64)])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("norm", [False, True])
def test_store_and_read(device, dtype, kept, width, rope, page, bits, norm):
    g = torch.Generator().manual_seed(width + rope + page + bits)
    tokens, pages = 77, 9
    kept = TYPES[kept]
    rows = normal(g, tokens, width + rope + 8, dtype=TYPES[dtype], size=3.0)
    latent, key = rows[:, :width], rows[:, width:width + rope]
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    slots[5], slots[9], slots[30] = -1, pages * page, -(1 << 31)
    positions = torch.randint(0, 100000, (tokens,), generator=g, dtype=torch.int32)
    weight = 1.0 + 0.3 * normal(g, width) if norm else None
    table, freqs = ops.rope_table(rope, 10000.0), plain.frequencies(rope, 10000.0)
    cache = ops.latent_cache(pages, page, width, rope, dtype=kept, bits=bits, device=device)
    for a in cache.values():
        a.view(torch.uint8).fill_(0x11)
    held = {k: v.clone() for k, v in cache.items()}
    layout = "half" if page == 48 else "interleaved"
    on = rows.to(device)
    ops.latent_store(cache, on[:, :width], on[:, width:width + rope], slots.to(device), positions.to(device), table, layout=layout, weight=None if weight is None else weight.to(device), eps=1e-5)
    real = (slots >= 0) & (slots < pages * page)
    # Slots that no row names keep what they had.
    named = torch.zeros(pages * page, dtype=torch.bool)
    named[slots[real].long()] = True
    for name, a in cache.items():
        flat = lambda t: t.cpu().flatten(0, 1)[~named].view(torch.uint8)  # noqa: E731
        assert torch.equal(flat(a), flat(held[name])), name
    got_latent, got_key = ops.latent_read(cache, slots.to(device), torch.float32)
    assert (got_latent[~real.to(device)] == 0).all() and (got_key[~real.to(device)] == 0).all()
    x = latent.double()
    if norm:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * weight.double()
    x, got_latent = x[real], got_latent.cpu()[real]
    # A normalised value: the squares' sum (9 roundings a lane and 6 over the lanes), the root and reciprocal, two products: 2^-20 in all.
    before = x.abs() * 2.0 ** -20 if norm else torch.zeros_like(x)
    if bits == 16:
        within(got_latent, x, before + x.abs() * plain.HALF[kept] * 1.01 + plain.LEAST[kept], "latent")
    elif not norm:
        codes, scales = plain.encode(latent.float()[real])
        flat = cache["latent"].cpu().view(-1, width)[slots[real].long()], cache["scale"].cpu().view(-1)[slots[real].long()]
        assert torch.equal(flat[0], codes) and torch.equal(flat[1], scales)
        assert torch.equal(got_latent.double(), plain.code_values(codes, scales))
    else:
        # Half an E4M3 step (2^-4 of the value, of the smallest normal one below it), or what the value's own error moves.
        scale = torch.exp2(cache["scale"].cpu().view(-1)[slots[real].long()].double() - 127.0)[:, None]
        assert (x.abs().amax(-1, keepdim=True) <= 448.0 * scale * (1 + 2.0 ** -19)).all()
        within(got_latent, x, before + torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10) * 1.001, "latent")
    want = plain.rotate(key[real], positions[real], freqs, layout)
    within(got_key.cpu()[real], want, rotation_bound(want, key[real].double(), torch.float32) + want.abs() * plain.HALF[kept] * 1.01 + plain.LEAST[kept], "key")
    # The same rows in the cache's own type: a rounding of the values.
    own = ops.latent_read(cache, slots.to(device))
    assert torch.equal(own[0].cpu()[real], got_latent.to(kept)) and torch.equal(own[1].cpu()[real], got_key.cpu()[real].to(kept))


def test_store_values_at_the_edges_of_eight_bits(device):
    """Rows of zeros, of the least and the largest numbers, infinities and NaN, and magnitudes of 448 times powers of two."""
    width = 256
    x = torch.zeros(10, width)
    x[1, 3] = 2.0 ** -149
    x[2, :4] = torch.tensor([3.4e38, -3.4e38, 1e30, -0.0])
    x[3, :3] = torch.tensor([math.inf, 1.0, -2.0])
    x[4, :3] = torch.tensor([math.nan, 448.0, -1.5])
    for i, e in enumerate((-20, 0, 1, 37)):
        x[5 + i] = torch.linspace(-448.0, 448.0, width) * 2.0 ** e
    x[9] = torch.linspace(-1, 1, width) * 2.0 ** -130
    cache = ops.latent_cache(1, 16, width, 32, bits=8, device=device)
    slots = torch.arange(10, dtype=torch.int32)
    ops.latent_store(cache, x.to(device), torch.zeros(10, 32, device=device), slots.to(device))
    codes, scales = plain.encode(x)
    got = cache["latent"].cpu()[0, :10], cache["scale"].cpu()[0, :10]
    assert torch.equal(got[1], scales)
    nan = torch.isnan(x)
    assert torch.equal(got[0][~nan], codes[~nan]) and ((got[0][nan] & 127) == 127).all()
    read = ops.latent_read(cache, slots.to(device), torch.float32)[0].cpu().double()
    want = plain.code_values(codes, scales)
    assert torch.equal(read[~nan], want[~nan].float().double()) and torch.isnan(read[nan]).all()


def test_store_without_rotation_and_one_token(device):
    g = torch.Generator().manual_seed(1)
    cache = ops.latent_cache(2, 16, 512, 64, dtype=torch.float16, device=device)
    x, key = normal(g, 1, 512, dtype=torch.float16).to(device), normal(g, 1, 64, dtype=torch.float16).to(device)
    ops.latent_store(cache, x, key, torch.tensor([17], dtype=torch.int32, device=device))
    assert torch.equal(cache["latent"][1, 1], x[0]) and torch.equal(cache["rope"][1, 1], key[0])
    ops.latent_store(cache, x[:0], key[:0], torch.empty(0, dtype=torch.int32, device=device))
    empty = ops.latent_read(cache, torch.empty(0, dtype=torch.int32, device=device))
    assert empty[0].shape == (0, 512) and empty[1].shape == (0, 64)


# ---------------------------------------------------------------- the heads' products


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,heads,k,n", [(1, 1, 32, 32), (1, 128, 128, 512), (31, 3, 512, 128), (33, 5, 96, 160), (64, 2, 64, 32), (65, 2, 160, 224), (129, 3, 512, 128), (300, 2, 128, 512),
                                              (200, 1, 32, 96)])
def test_project(device, dtype, tokens, heads, k, n):
    g = torch.Generator().manual_seed(tokens + k + n)
    x, w = normal(g, tokens, heads, k, dtype=TYPES[dtype]), normal(g, heads, n, k, dtype=TYPES[dtype])
    got = ops.latent_project(x.to(device), w.to(device))
    want = torch.einsum("thk,hnk->thn", x.double(), w.double())
    size = torch.einsum("thk,hnk->thn", x.double().abs(), w.double().abs())
    bound = size * k * 2.0 ** -24
    within(got, want, bound + (want.abs() + bound) * plain.HALF[TYPES[dtype]] * 1.01 + plain.LEAST[TYPES[dtype]])


@pytest.mark.parametrize("tokens", [3, 70])
def test_project_strides(device, tokens):
    """Views: a part of every head's query, the value rows of one expansion matrix, a part of a wider result."""
    g = torch.Generator().manual_seed(tokens)
    q, expand = normal(g, tokens, 7, 192, dtype=torch.bfloat16).to(device), normal(g, 4, 96 + 128, 256, dtype=torch.bfloat16).to(device)
    wide = torch.full((tokens, 4, 200), 7.0, dtype=torch.bfloat16, device=device)
    x = normal(g, tokens, 6, 256, dtype=torch.bfloat16).to(device)[:, 1:5]
    ops.latent_project(x, expand[:, 96:], out=wide[..., 8:136])
    want = torch.einsum("thk,hnk->thn", x.double().cpu(), expand[:, 96:].double().cpu())
    within(wide[..., 8:136], want, 256 * 256 * 2.0 ** -22 + want.abs() * 2.0 ** -8 * 1.01)
    assert (wide[..., :8] == 7).all() and (wide[..., 136:] == 7).all()
    turned = expand[:, :64, :].transpose(1, 2).contiguous()  # a copy made once: [heads, 256, 64]
    got = ops.latent_project(q[:, :4, 128:], turned)
    want = torch.einsum("thk,hkn->thn", q[:, :4, 128:].double().cpu(), expand[:, :64].double().cpu())
    within(got, want, 64 * 64 * 2.0 ** -22 + want.abs() * 2.0 ** -8 * 1.01)


# ---------------------------------------------------------------- the absorbed form


def latent_case(g, lengths, new, page, heads, width, rope, dtype, bits, extra=2):
    """A cache whose unnamed places hold NaN, a table in any order, and queries."""
    dtype = TYPES[dtype]
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + extra
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(held) + 1), -1, dtype=torch.int32)
    latent, key = torch.full((pages, page, width), math.nan), torch.full((pages, page, rope), math.nan, dtype=dtype)
    codes, scales = torch.full((pages, page, width), 0x7F, dtype=torch.uint8), torch.full((pages, page), 0xFF, dtype=torch.uint8)
    at = 0
    for r, n in enumerate(lengths):
        for j in range(held[r]):
            p = int(order[at])
            at += 1
            table[r, j] = p
            count = min(page, n - j * page)
            latent[p, :count] = torch.randn(count, width, generator=g)
            key[p, :count] = torch.randn(count, rope, generator=g).to(dtype)
            if bits == 8:
                codes[p, :count] = torch.randint(0, 256, (count, width), generator=g).to(torch.uint8)
                codes[p, :count][(codes[p, :count] & 127) == 127] = 0
                scales[p, :count] = torch.randint(114, 121, (count,), generator=g).to(torch.uint8)
    cache = {"latent": latent.to(dtype), "rope": key} if bits == 16 else {"latent": codes, "scale": scales, "rope": key}
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    tokens = starts[-1] + 1  # a row behind the last request's
    q_latent, q_rope = normal(g, tokens, heads, width, dtype=dtype, size=1.0), normal(g, tokens, heads, rope, dtype=dtype)
    return cache, table, starts, q_latent, q_rope


def cache_values(cache):
    return plain.code_values(cache["latent"], cache["scale"]) if "scale" in cache else cache["latent"].double()


def check_attend(device, cache, table, lengths, starts, q_latent, q_rope, scale, before=None, most=None):
    """Every row against its definition; rows behind the last request's stay as they are."""
    dtype = q_latent.dtype
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    out = torch.full(q_latent.shape, 55.0, dtype=dtype, device=device)
    on = {k: v.to(device) for k, v in cache.items()}
    ops.latent_attend(on, q_latent.to(device), q_rope.to(device), table.to(device), ints(lengths), ints(starts), scale, before=None if before is None else ints(before), most=most, out=out)
    got = out.cpu()
    values, pages, page = cache_values(cache), cache["rope"].shape[0], cache["rope"].shape[1]
    heads = q_latent.shape[1]
    for r, length in enumerate(lengths):
        n = starts[r + 1] - starts[r]
        if n <= 0:
            continue
        entries = table[r, :-(-length // page)].long()
        there = (entries >= 0) & (entries < pages)
        c = values[entries.clamp(0, pages - 1)].reshape(-1, values.shape[2])[:length]
        k = torch.cat([c, cache["rope"][entries.clamp(0, pages - 1)].double().reshape(-1, q_rope.shape[2])[:length]], 1)
        first = before[r] if before is not None else length - n
        rows = slice(starts[r], starts[r + 1])
        q = torch.cat([q_latent[rows], q_rope[rows]], -1).double().reshape(n * heads, -1)
        position = (first + torch.arange(n)).repeat_interleave(heads)
        want, size, logits = plain.attention(q, k, c, scale, position, there.repeat_interleave(page)[:length])
        plain.close(got[rows].reshape(n * heads, -1), want, size, logits, dtype, k.shape[1], max(length, 1))
    assert (got[starts[-1]:] == 55.0).all()


SHAPES = [  # lengths, new tokens, page, heads, most
    ([1], [1], 16, 1, 1), ([5], [1], 16, 16, 1), ([33, 64, 1, 32, 31], [1, 1, 1, 0, 1], 16, 16, 1), ([700, 3, 257, 90], [1, 1, 1, 1], 48, 7, 1),
    ([100, 2, 61], [3, 2, 1], 16, 5, 3), ([300, 40], [1, 1], 64, 128, 1), ([90, 35], [1, 1], 32, 40, 1), ([130, 77], [2, 2], 16, 160, 2),
    ([64, 200, 37], [64, 30, 37], 16, 3, 64), ([50], [50], 256, 33, 50), ([1500], [1], 128, 16, 1), ([1300, 1], [1, 1], 128, 129, 1)]


@pytest.mark.parametrize("lengths,new,page,heads,most", SHAPES)
@pytest.mark.parametrize("width,rope,dtype,bits", [(512, 64, "bf16", 16), (512, 64, "bf16", 8), (256, 32, "f16", 16), (256, 64, "f16", 8), (512, 32, "f16", 16), (512, 32, "f16", 8),
                                                   (256, 32, "bf16", 8), (256, 64, "bf16", 16)])
def test_attend(device, lengths, new, page, heads, most, width, rope, dtype, bits):
    g = torch.Generator().manual_seed(sum(lengths) + heads + width + bits)
    cache, table, starts, q_latent, q_rope = latent_case(g, lengths, new, page, heads, width, rope, dtype, bits)
    check_attend(device, cache, table, lengths, starts, q_latent, q_rope, (0.2 if bits == 8 else 1.5) / math.sqrt(width + rope), most=most)
    if heads == 5:
        check_attend(device, cache, table, lengths, starts, q_latent, q_rope, -0.05, most=None)
        check_attend(device, cache, table, lengths, starts, q_latent, q_rope, 0.0, most=None)


# ---------------------------------------------------------------- the expanded form


def check_prompt(device, q, k, k_rope, v, starts, key_starts, scale, most=None):
    ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    dtype = q.dtype
    out = torch.full((q.shape[0], q.shape[1], v.shape[2]), 55.0, dtype=dtype, device=device)
    ops.latent_prompt(q.to(device), k.to(device), k_rope.to(device), v.to(device), ints(starts), scale, key_starts=ints(key_starts), most=most, out=out)
    got = out.cpu()
    keys = starts if key_starts is None else key_starts
    for r in range(len(starts) - 1):
        n, m = starts[r + 1] - starts[r], keys[r + 1] - keys[r]
        rows, at = slice(starts[r], starts[r + 1]), slice(keys[r], keys[r + 1])
        for h in range(q.shape[1]):
            want, size, logits = plain.attention(q[rows, h].double(), torch.cat([k[at, h], k_rope[at]], 1).double(), v[at, h].double(), scale,
                                                 torch.arange(m - n, m), torch.ones(m, dtype=torch.bool))
            plain.close(got[rows, h], want, size, logits, dtype, q.shape[2], max(m, 1))
    assert (got[starts[-1]:] == 55.0).all()


@pytest.mark.parametrize("new,keys,heads,most", [([1], None, 1, None), ([1], [1], 3, 1), ([64], None, 2, 64), ([129], [300], 2, None), ([5, 0, 40, 1], [70, 9, 40, 65], 3, 40),
                                                 ([3], [2000], 2, 3), ([127, 2], [127, 800], 5, 127), ([7, 3], [4, 0], 2, 7)])
@pytest.mark.parametrize("nope,rope,value,dtype", [(128, 64, 128, "bf16"), (64, 32, 64, "f16"), (64, 64, 64, "bf16"), (128, 32, 128, "f16"), (64, 64, 128, "bf16"), (128, 32, 64, "f16"), (128, 64, 64, "bf16"),
                                                   (64, 32, 128, "f16")])
def test_prompt(device, new, keys, heads, most, nope, rope, value, dtype):
    g = torch.Generator().manual_seed(sum(new) + heads + nope)
    add = lambda v: [sum(v[:i]) for i in range(len(v) + 1)]  # noqa: E731
    starts, key_starts = add(new), None if keys is None else add(keys)
    count = starts[-1] if keys is None else key_starts[-1]
    dtype = TYPES[dtype]
    q = normal(g, starts[-1] + 2, heads, nope + rope, dtype=dtype, size=1.5)
    kv = normal(g, count, heads, nope + value + 8, dtype=dtype)
    k_rope = normal(g, count, rope + 16, dtype=dtype)[:, 8:8 + rope]
    check_prompt(device, q, kv[..., :nope], k_rope, kv[..., nope:nope + value], starts, key_starts, 1.0 / math.sqrt(nope + rope), most)
