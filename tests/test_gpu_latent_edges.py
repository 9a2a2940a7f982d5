"""Attention over latent vectors where it can go wrong: what rows must not see, pages that are missing, more tokens than pages, many requests, views, long caches, other
streams, captured launches that replay at other lengths, and the operators together as a layer runs them."""
import math

import pytest
import torch

import latent_plain as plain
from llmp_amd import ops
from test_gpu_latent import TYPES, cache_values, check_attend, check_prompt, latent_case, normal, within

pytestmark = pytest.mark.gpu

GARBAGE = [math.nan, math.inf, -math.inf]


def ints(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def attend(device, cache, table, lengths, starts, q_latent, q_rope, scale, **kw):
    on = {k: v.to(device) for k, v in cache.items()}
    return ops.latent_attend(on, q_latent.to(device), q_rope.to(device), table.to(device), ints(lengths, device), ints(starts, device), scale, **kw).cpu()


# ---------------------------------------------------------------- what a row must not see


@pytest.mark.parametrize("heads", [3, 16, 48])
@pytest.mark.parametrize("width,rope,dtype,bits", [(512, 64, "bf16", 16), (512, 64, "bf16", 8), (256, 32, "f16", 16), (256, 64, "bf16", 8)])
def test_later_tokens_of_infinities_and_nan(device, heads, width, rope, dtype, bits):
    """The last tokens hold what is no number (a value, a whole row, a rotated key, a scale): rows before them are as if they were not there, rows that see them are no
    numbers where a value is none."""
    g = torch.Generator().manual_seed(heads + width + bits)
    lengths, new = [37, 70, 6], [5, 33, 6]
    cache, table, starts, q_latent, q_rope = latent_case(g, lengths, new, 16, heads, width, rope, dtype, bits)
    scale = 0.02
    clean = attend(device, cache, table, lengths, starts, q_latent, q_rope, scale)
    for r, length in enumerate(lengths):
        for back, kind in ((1, 0), (2, 1), (3, 2)):
            p = length - back
            page, at = int(table[r, p // 16]), p % 16
            if bits == 8:
                cache["latent"][page, at, ::3] = 0x7F if kind != 1 else 0xFF
            else:
                cache["latent"][page, at, ::3] = GARBAGE[kind]
            if kind == 2:
                cache["rope"][page, at, 1] = GARBAGE[kind]
    got = attend(device, cache, table, lengths, starts, q_latent, q_rope, scale)
    for r, n in enumerate(new):
        keeps = slice(starts[r], starts[r + 1] - 3)
        # (The same sums of the same values: bit for bit.)
        assert torch.equal(got[keeps], clean[keeps]), r
        assert not torch.isfinite(got[starts[r + 1] - 1][:, ::3].float()).any(), r


@pytest.mark.parametrize("width", [512, 256])
def test_rows_that_see_infinities_give_the_same_bits_again(device, width):
    """Rows that see a token of infinities whose logit is the lowest, beside rows that must not see it."""
    g = torch.Generator().manual_seed(width)
    cache, table, starts, q_latent, q_rope = latent_case(g, [90], [33], 16, 48, width, 64, "bf16", 16)
    page, at = int(table[0, 75 // 16]), 75 % 16
    cache["latent"][page, at] = 0.0
    cache["latent"][page, at, 5] = math.inf
    q_latent[..., 5] = -q_latent[..., 5].abs() - 0.5
    first = attend(device, cache, table, [90], starts, q_latent, q_rope, 0.02)
    for _ in range(5):
        again = attend(device, cache, table, [90], starts, q_latent, q_rope, 0.02)
        assert torch.equal(first[:33].view(torch.int16), again[:33].view(torch.int16))


@pytest.mark.parametrize("heads,most", [(8, 1), (16, 1), (128, 1), (20, 9)])
@pytest.mark.parametrize("bits", [16, 8])
def test_pages_that_are_missing(device, heads, most, bits):
    """Entries that are no page, at the beginning, in the middle, for all that a request holds: their tokens change nothing, a row that sees none is zero."""
    g = torch.Generator().manual_seed(heads + bits)
    lengths, new = [200, 90, 33, 500], [min(most, 9), 1, min(most, 4), most]
    cache, table, starts, q_latent, q_rope = latent_case(g, lengths, new, 32, heads, 512, 64, "bf16", bits)
    pages = cache["rope"].shape[0]
    table[0, 0], table[0, 3], table[0, 4] = -1, pages, (1 << 31) - 1
    table[1, :] = -(1 << 31)
    table[2, 1] = -7
    table[3, 5:12] = pages + 3
    check_attend(device, cache, table, lengths, starts, q_latent, q_rope, 0.03, most=most)
    out = attend(device, cache, table, lengths, starts, q_latent, q_rope, 0.03, most=most)
    assert (out[starts[1]:starts[2]] == 0).all()


@pytest.mark.parametrize("heads", [4, 40])
def test_a_step_whose_pages_ran_out(device, heads):
    """`before` and lengths that end before a request's new tokens: a token past what is held keeps its position and sees all that is held; none held: zero."""
    g = torch.Generator().manual_seed(heads)
    lengths, new, before = [40, 17, 0, 64], [6, 4, 3, 2], [38, 17, 0, 62]
    cache, table, starts, q_latent, q_rope = latent_case(g, lengths, new, 16, heads, 256, 64, "bf16", 16)
    check_attend(device, cache, table, lengths, starts, q_latent, q_rope, 0.04, before=before)


def test_lengths_shorter_than_the_new_tokens(device):
    """Without `before` the first of them lie before position 0: they see nothing."""
    g = torch.Generator().manual_seed(9)
    for heads in (2, 32):
        lengths, new = [3, 20], [7, 2]
        cache, table, starts, q_latent, q_rope = latent_case(g, lengths, new, 16, heads, 512, 32, "f16", 16)
        check_attend(device, cache, table, lengths, starts, q_latent, q_rope, 0.04)


@pytest.mark.parametrize("heads", [1, 16, 24])
def test_more_requests_than_a_wave_has_lanes(device, heads):
    g = torch.Generator().manual_seed(heads)
    lengths = torch.randint(0, 80, (150,), generator=g).tolist()
    lengths[70] = 900
    new = [min(n, 1) for n in lengths]
    cache, table, starts, q_latent, q_rope = latent_case(g, lengths, new, 16, heads, 256, 32, "bf16", 8)
    check_attend(device, cache, table, lengths, starts, q_latent, q_rope, 0.02, most=1)


def test_tables_shorter_than_lengths(device):
    """A table row of fewer pages than a length needs: the tokens behind it are not there."""
    g = torch.Generator().manual_seed(4)
    cache, table, starts, q_latent, q_rope = latent_case(g, [100, 40], [1, 1], 16, 16, 512, 64, "bf16", 16)
    got = attend(device, cache, table[:, :4].contiguous(), [100, 40], starts, q_latent, q_rope, 0.05, most=1)
    want = attend(device, cache, table[:, :4].contiguous(), [64, 40], starts, q_latent, q_rope, 0.05, most=1)
    assert torch.equal(got[:2], want[:2])


# ---------------------------------------------------------------- views, far slots


def test_queries_and_results_that_are_views(device):
    """The rotated part as the end of whole heads, every other head of a wider latent query, results among other values, a table that is part of a wider one."""
    g = torch.Generator().manual_seed(12)
    for heads, most in ((8, 1), (30, 3)):
        lengths, new = [75, 130], [1, most]
        cache, table, starts, q_latent, q_rope = latent_case(g, lengths, new, 16, heads, 256, 64, "f16", 16)
        tokens = starts[-1]
        plainly = attend(device, cache, table, lengths, starts, q_latent[:tokens], q_rope[:tokens], 0.05, most=most)
        wide = torch.randn(tokens, 2 * heads, 256 + 8, device=device).half()
        whole = torch.randn(tokens, heads, 192, device=device).half()
        wide[:, ::2, 8:] = q_latent[:tokens].to(device)
        whole[..., 128:] = q_rope[:tokens].to(device)
        tables = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device=device)
        tables[:, :table.shape[1]] = table.to(device)
        out = torch.full((tokens, heads + 2, 264), 3.0, dtype=torch.float16, device=device)
        on = {k: v.to(device) for k, v in cache.items()}
        ops.latent_attend(on, wide[:, ::2, 8:], whole[..., 128:], tables[:, :table.shape[1]], ints(lengths, device), ints(starts, device), 0.05, most=most, out=out[:, 1:-1, :256])
        assert torch.equal(out[:, 1:-1, :256].cpu(), plainly)
        assert (out[:, 0] == 3).all() and (out[:, -1] == 3).all() and (out[..., 256:] == 3).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_a_cache_of_more_than_four_gib(device, bits):
    """Slots whose bytes lie past 2^32 (16 bits: 2^23 tokens of 1024 bytes): stored, read and attended as they are near the beginning."""
    g = torch.Generator().manual_seed(bits)
    page, pages = 256, (1 << 23) // 256 if bits == 16 else (1 << 24) // 256
    cache = {"latent": torch.empty((pages, page, 512), dtype=torch.bfloat16 if bits == 16 else torch.uint8, device=device), "rope": torch.empty((pages, page, 64), dtype=torch.bfloat16, device=device)}
    if bits == 8:
        cache["scale"] = torch.empty((pages, page), dtype=torch.uint8, device=device)
    small = ops.latent_cache(4, page, 512, 64, bits=bits, device=device)
    far = [pages - 1, 2, pages // 2 + 1, pages - 2]
    x, key = normal(g, 900, 512, dtype=torch.bfloat16).to(device), normal(g, 900, 64, dtype=torch.bfloat16).to(device)
    at = torch.arange(900, dtype=torch.int32)
    slots = torch.tensor(far, dtype=torch.int32)[at // page] * page + at % page
    table = ops.rope_table(64)
    ops.latent_store(cache, x, key, slots.to(device), at.to(device), table)
    ops.latent_store(small, x, key, at.to(device), at.to(device), table)
    for a, b in zip(ops.latent_read(cache, slots.to(device)), ops.latent_read(small, at.to(device))):
        assert torch.equal(a, b)
    for heads in (16, 64):
        q, r = normal(g, 1, heads, 512, dtype=torch.bfloat16).to(device), normal(g, 1, heads, 64, dtype=torch.bfloat16).to(device)
        outs = [ops.latent_attend(c, q, r, ints([pages_], device), ints([900], device), ints([0, 1], device), 0.05, most=1) for c, pages_ in ((cache, far), (small, [0, 1, 2, 3]))]
        assert torch.equal(*outs)


# ---------------------------------------------------------------- the expanded form


@pytest.mark.parametrize("dtype,nope,rope,value", [("bf16", 128, 64, 128), ("f16", 64, 32, 64), ("bf16", 64, 64, 128), ("f16", 128, 32, 64)])
def test_prompt_later_values_of_infinities_and_nan(device, dtype, nope, rope, value):
    """Keys and values that only later rows see, and those of other requests."""
    g = torch.Generator().manual_seed(nope)
    starts, key_starts, heads = [0, 70, 140, 141], [0, 70, 290, 300], 3
    q, k = normal(g, 141, heads, nope + rope, dtype=TYPES[dtype]), normal(g, 300, heads, nope, dtype=TYPES[dtype])
    v, k_rope = normal(g, 300, heads, value, dtype=TYPES[dtype]), normal(g, 300, rope, dtype=TYPES[dtype])

    def run():
        return ops.latent_prompt(q.to(device), k.to(device), k_rope.to(device), v.to(device), ints(starts, device), 0.05, key_starts=ints(key_starts, device)).cpu()

    clean = run()
    for j, bad in ((69, 0), (289, 1), (288, 2), (68, 1)):
        v[j, :, ::2] = GARBAGE[bad]
    k[289, 1], k_rope[69, 3], k[299] = math.nan, math.inf, math.nan
    got = run()
    for rows in (slice(0, 68), slice(70, 138)):
        assert torch.equal(got[rows], clean[rows])
    assert not torch.isfinite(got[69][:, ::2].float()).any() and not torch.isfinite(got[139][:, ::2].float()).any() and torch.isnan(got[140].float()).all()


@pytest.mark.parametrize("heads,new,keys,nope,rope,value", [(64, [1100], None, 128, 64, 128), (64, [1100], None, 64, 32, 64), (128, [300, 700, 5], [900, 700, 1200], 64, 64, 64),
                                                            (64, [1100], None, 64, 64, 128), (64, [1100], None, 128, 32, 64)])
def test_prompt_of_whole_pairs(device, heads, new, keys, nope, rope, value):
    """Where rows are many a workgroup takes all keys of its rows; three heads of them are checked."""
    g = torch.Generator().manual_seed(heads + sum(new))
    add = lambda v: [sum(v[:i]) for i in range(len(v) + 1)]  # noqa: E731
    starts, key_starts = add(new), add(keys or new)
    dtype = torch.bfloat16
    q, k, v = (normal(g, n, heads, d, dtype=dtype) for n, d in ((starts[-1], nope + rope), (key_starts[-1], nope), (key_starts[-1], value)))
    k_rope = normal(g, key_starts[-1], rope, dtype=dtype)
    got = ops.latent_prompt(q.to(device), k.to(device), k_rope.to(device), v.to(device), ints(starts, device), 0.08, key_starts=None if keys is None else ints(key_starts, device), most=max(new)).cpu()
    for r in range(len(new)):
        n, m = new[r], key_starts[r + 1] - key_starts[r]
        picked = torch.unique(torch.cat([torch.arange(0, n, 97), torch.tensor([n - 1])]))
        for h in (0, heads // 2 + 1, heads - 1):
            at = slice(key_starts[r], key_starts[r + 1])
            want, size, logits = plain.attention(q[starts[r] + picked, h].double(), torch.cat([k[at, h], k_rope[at]], 1).double(), v[at, h].double(), 0.08, m - n + picked, torch.ones(m, dtype=torch.bool))
            plain.close(got[starts[r] + picked, h], want, size, logits, dtype, nope + rope, m)


def test_prompt_of_many_requests_and_a_first_row_further_on(device):
    g = torch.Generator().manual_seed(21)
    new = torch.randint(0, 9, (90,), generator=g).tolist()
    more = torch.randint(0, 60, (90,), generator=g).tolist()
    keys = [n + m for n, m in zip(new, more)]
    starts = [3 + sum(new[:i]) for i in range(91)]
    key_starts = [5 + sum(keys[:i]) for i in range(91)]
    q = normal(g, starts[-1] + 1, 2, 96, dtype=torch.float16)
    k, v, k_rope = normal(g, key_starts[-1] + 2, 2, 64, dtype=torch.float16), normal(g, key_starts[-1] + 2, 2, 64, dtype=torch.float16), normal(g, key_starts[-1] + 2, 32, dtype=torch.float16)
    check_prompt(device, q, k, k_rope, v, starts, key_starts, 0.1, most=8)


def test_prompt_without_any_keys(device):
    q, none, starts = torch.randn(5, 3, 192, device=device).bfloat16(), torch.empty(0, 3, 128, dtype=torch.bfloat16, device=device), ints([0, 2, 5], device)
    out = torch.full((5, 3, 128), 9.0, dtype=torch.bfloat16, device=device)
    ops.latent_prompt(q, none, torch.empty(0, 64, dtype=torch.bfloat16, device=device), none, starts, 0.1, key_starts=ints([0, 0, 0], device), out=out)
    assert (out == 0).all()


def test_prompt_of_many_requests_without_a_bound(device):
    """No word of how many queries a request has: 600 prompts of a few tokens."""
    g = torch.Generator().manual_seed(22)
    new = torch.randint(0, 7, (600,), generator=g).tolist()
    starts = [sum(new[:i]) for i in range(601)]
    q, k, v, k_rope = (normal(g, starts[-1], *s, dtype=torch.bfloat16) for s in ((2, 192), (2, 128), (2, 128), (64,)))
    check_prompt(device, q, k, k_rope, v, starts, None, 0.1, most=None)


# ---------------------------------------------------------------- streams and graphs


def step_inputs(device, heads, bits=16, seed=2):
    g = torch.Generator().manual_seed(seed)
    lengths = [700, 90, 300]
    cache, table, starts, q_latent, q_rope = latent_case(g, lengths, [1, 1, 1], 16, heads, 512, 64, "bf16", bits)
    return ({k: v.to(device) for k, v in cache.items()}, table.to(device), ints(lengths, device), ints(starts, device), q_latent[:3].to(device), q_rope[:3].to(device))


def test_the_same_bits_again_and_on_another_stream(device):
    for heads in (16, 128):
        cache, table, n, starts, q, r = step_inputs(device, heads)
        first = ops.latent_attend(cache, q, r, table, n, starts, 0.05, most=1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = [ops.latent_attend(cache, q, r, table, n, starts, 0.05, most=1) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(first, a) for a in again)


@pytest.mark.parametrize("heads,bits", [(16, 16), (16, 8), (128, 16)])
def test_captured_steps_replay_at_other_lengths(device, heads, bits):
    """Rotation, store, query product, attention and the product back in one graph, replayed over other lengths, positions and values, with eager work in between."""
    cache, table, n, starts, _, _ = step_inputs(device, heads, bits)
    g = torch.Generator().manual_seed(7)
    turns = ops.rope_table(64)
    new = lambda *shape: normal(g, *shape, dtype=torch.bfloat16).to(device)  # noqa: E731
    q, rows, up, down = new(3, heads, 128 + 64), new(3, 512 + 64), new(heads, 512, 128), new(heads, 128, 512)
    weight = torch.ones(512, device=device)
    positions, slots = ints([699, 89, 299], device), ints([0, 0, 0], device)
    scratch = torch.empty(256 << 20, dtype=torch.uint8, device=device)

    def work():
        turned = ops.rope(q, positions, turns, first=128)
        ops.latent_store(cache, rows[:, :512], rows[:, 512:], slots, positions, turns, weight=weight)
        over = ops.latent_attend(cache, ops.latent_project(turned[..., :128], up), turned[..., 128:], table, n, starts, 0.03, most=1, scratch=scratch)
        return ops.latent_project(over, down)

    def at(lengths):
        n.copy_(ints(lengths, device))
        positions.copy_(n - 1)
        slots.copy_(torch.stack([table[i, (m - 1) // 16] * 16 + (m - 1) % 16 for i, m in enumerate(lengths)]))
        q.copy_(new(3, heads, 192))
        rows.copy_(new(3, 576))

    at([700, 90, 300])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for lengths in ([700, 90, 300], [1, 64, 33], [512, 1, 2], [699, 89, 17]):
        at(lengths)
        want = work().clone()
        torch.cuda.synchronize()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), lengths
            out.zero_()


def test_two_graphs_on_one_workspace(device):
    """One after the other on a stream, in either order: nothing of a launch is in the workspace before it."""
    cache, table, n, starts, q, r = step_inputs(device, 16)
    g = torch.Generator().manual_seed(8)
    p = [normal(g, *s, dtype=torch.bfloat16).to(device) for s in ((40, 2, 192), (2000, 2, 128), (2000, 64), (2000, 2, 128))]
    rows, keys = ints([0, 40], device), ints([0, 2000], device)
    scratch = torch.empty(256 << 20, dtype=torch.uint8, device=device)
    works = [lambda: ops.latent_attend(cache, q, r, table, n, starts, 0.05, most=1, scratch=scratch),
             lambda: ops.latent_prompt(*p, rows, 0.05, key_starts=keys, most=40, scratch=scratch)]
    want = [w().clone() for w in works]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for w in works:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(w())
    scratch.fill_(0xFF)
    for order in ((0, 1), (1, 0), (1, 1), (0, 0)):
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in set(order):
            assert torch.equal(outs[i], want[i]), order
            outs[i].zero_()


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("heads,bits", [(16, 16), (40, 16), (16, 8)])
def test_a_layer_in_both_forms(device, heads, bits):
    """Two requests' prompts (rotation, store, what the cache gives back made into heads' keys and values, the expanded form), then the same rows by the absorbed form: query
    products, attention over the cache, products back. Both against the layer's definition over what the cache holds."""
    g = torch.Generator().manual_seed(heads + bits)
    dtype, width, nope, rope, page = torch.bfloat16, 512, 128, 64, 16
    new = [37, 90]
    starts = [0, 37, 127]
    tokens = 127
    cache = ops.latent_cache(12, page, width, rope, bits=bits, device=device)
    table = torch.tensor([[7, 2, 9, -1, -1, -1], [0, 11, 3, 4, 8, 1]], dtype=torch.int32, device=device)
    positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in new]).to(device)
    owner = torch.tensor([0] * 37 + [1] * 90, device=device)
    slots = (table[owner, (positions // page).long()] * page + positions % page).to(torch.int32)
    turns = ops.rope_table(rope)
    q, rows = normal(g, tokens, heads, nope + rope, dtype=dtype).to(device), normal(g, tokens, width + rope, dtype=dtype, size=2.0).to(device)
    expand = normal(g, heads, 2 * nope, width, dtype=dtype, size=width ** -0.5).to(device)  # a head's keys, then its values, from the latent vector
    scale = 0.3 / math.sqrt(nope + rope)
    # As a program runs it.
    q = ops.rope(q, positions, turns, first=nope)
    ops.latent_store(cache, rows[:, :width], rows[:, width:], slots, positions, turns, weight=torch.ones(width, device=device))
    latent, k_rope = ops.latent_read(cache, slots)
    wide = ops.latent_project(latent[:, None].expand(-1, heads, -1), expand)
    expanded = ops.latent_prompt(q, wide[..., :nope], k_rope, wide[..., nope:], ints(starts, device), scale, most=90)
    up = expand[:, :nope].transpose(1, 2).contiguous()
    over = ops.latent_attend(cache, ops.latent_project(q[..., :nope], up), q[..., nope:], table, ints(new, device), ints(starts, device), scale, most=90)
    absorbed = ops.latent_project(over, expand[:, nope:])
    # The definition, over the held vectors.
    c, kr, q, w = latent.double().cpu(), k_rope.double().cpu(), q.double().cpu(), expand.double().cpu()
    k, v = torch.einsum("tc,hnc->thn", c, w[:, :nope]), torch.einsum("tc,hnc->thn", c, w[:, nope:])
    k_size, v_size = (torch.einsum("tc,hnc->thn", c.abs(), m.abs()) for m in (w[:, :nope], w[:, nope:]))
    half = 2.0 ** -8
    for r in range(2):
        at = slice(starts[r], starts[r + 1])
        causal = torch.tril(torch.ones(new[r], new[r], dtype=torch.bool))
        for h in range(heads):
            logits = (q[at, h, :nope] @ k[at, h].T + q[at, h, nope:] @ kr[at].T) * scale
            p = torch.softmax(torch.where(causal, logits, -math.inf), -1)
            want = p @ v[at, h]
            # A logit: the rounding of its keys or of its latent query, 2^-8 of the products' sizes, and F32 sums, less than that again by far; it moves weights and
            # their sum. Then the weights' rounding, the values' or the latent result's, of the products' sizes, and the result's.
            off = (q[at, h, :nope].abs() @ k_size[at, h].T * scale * half * 1.05).amax(1, keepdim=True)
            size = p @ v_size[at, h]
            bound = size * (2.0 * torch.expm1(2.0 * off) + 2.0 * half) * 1.05 + want.abs() * half * 1.05
            within(expanded[at, h], want, bound, f"expanded {r} {h}")
            within(absorbed[at, h], want, bound, f"absorbed {r} {h}")


def test_answers_token_by_token(device):
    """A plan's slots, a store and an attention a step, as requests grow: each step's rows against the definition over what the cache gives back."""
    g = torch.Generator().manual_seed(31)
    heads, width, rope, page, requests = 6, 256, 32, 16, 4
    dtype = torch.float16
    cache = ops.latent_cache(24, page, width, rope, dtype=dtype, device=device)
    table = torch.full((requests, 8), -1, dtype=torch.int32, device=device)
    ring, counters = torch.arange(24, dtype=torch.int32, device=device), ints([0, 24, 0], device)
    held, turns = [0] * requests, ops.rope_table(rope)
    for step in ([30, 1, 0, 17], [1, 1, 50, 1], [1, -1, 1, 2], [2, 20, 1, 1]):
        after = [0 if s < 0 else held[r] + s for r, s in enumerate(step)]
        rows = sum(max(a - b, 0) for a, b in zip(after, held))
        before = ints(held, device)
        plan = ops.paged_plan(before, ints(after, device), table, ring, counters, page, rows)
        counters = plan["counters"]
        x, q = normal(g, rows, width + rope, dtype=dtype).to(device), normal(g, rows, heads, width, dtype=dtype).to(device)
        qr = normal(g, rows, heads, rope, dtype=dtype).to(device)
        ops.latent_store(cache, x[:, :width], x[:, width:], plan["slots"], plan["positions"], turns)
        ops.rope(qr, plan["positions"], turns, out=qr)
        got = ops.latent_attend(cache, q, qr, table, plan["lengths"], plan["starts"], 0.05, before=before, most=max(max(step), 1))
        starts, lengths = plan["starts"].tolist(), plan["lengths"].tolist()
        assert lengths == after
        kept = {k: v.cpu() for k, v in cache.items()}
        values, names = cache_values(kept), table.cpu()
        for r in range(requests):
            n = starts[r + 1] - starts[r]
            if n == 0:
                continue
            entries = names[r, :-(-after[r] // page)].long()
            c = values[entries].reshape(-1, width)[:after[r]]
            k = torch.cat([c, kept["rope"][entries].double().reshape(-1, rope)[:after[r]]], 1)
            at = slice(starts[r], starts[r + 1])
            want, size, logits = plain.attention(torch.cat([q[at], qr[at]], -1).double().cpu().reshape(n * heads, -1), k, c, 0.05, (after[r] - n + torch.arange(n)).repeat_interleave(heads),
                                                 torch.ones(after[r], dtype=torch.bool))
            plain.close(got[at].reshape(n * heads, -1), want, size, logits, dtype, width + rope, after[r])
        held = after
