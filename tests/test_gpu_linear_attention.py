"""GPU checks of linear attention with a decay for each head against float64."""
import pytest
import torch

from linear64 import bounds, linear64
from vllm_exact.linear_attn import linear_attention_torch, linear_prompt, linear_step

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # the output's own rounding
LENS = [(1,), (0, 5, 0, 33), (31, 32, 63, 64, 65), (127, 129), (511, 513, 2), (1100,)]


def inputs(lens, H, KV, D, dtype, seed=0, extra=0, fused=False, magnitude=1.0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + extra
    x = torch.randn(T, H + 2 * KV, D, generator=g) * magnitude
    x[:, :, 3 % D] *= 4
    x = x.to(dtype).to(DEV)
    q, k, v = x.split((H, KV, KV), dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    return q, k, v, ints([0] + list(lens)).cumsum(0).to(torch.int32)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def decays(H, kind="windows"):
    if kind == "windows":
        return (-(2.0 ** (-8.0 * (torch.arange(H) + 1) / H))).to(DEV)
    return torch.tensor([0.0, -float("inf"), -50.0, -1e-3, -3.0])[torch.arange(H) % 5].to(DEV)


def check(got, want, bound, dtype=torch.float32):
    err = (got.double() - want).abs()
    room = bound + want.abs() * HALF[dtype] + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133)
    assert torch.isfinite(got).all()
    assert (err <= room).all(), f"off by {float((err / room.clamp(min=1e-300)).max())} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,KV,D", [(1, 1, 64), (4, 2, 128), (2, 1, 256), (5, 5, 64)])
@pytest.mark.parametrize("lens", LENS)
def test_prompts_from_zeros(lens, H, KV, D, dtype):
    q, k, v, cu = inputs(lens, H, KV, D, dtype, extra=3)
    g, scale = decays(H), D ** -0.5
    out = torch.full((len(q), H, D), 7.0, device=DEV, dtype=dtype)
    state = torch.full((len(lens) + 2, H, D, D), 9.0, device=DEV)
    slots = torch.randperm(len(lens) + 2, generator=torch.Generator().manual_seed(1))[:len(lens)]
    assert linear_prompt(q, k, v, cu, g, scale, out, state, None, slots.to(torch.int32).to(DEV)) is out
    want, ends = linear64(q, k, v, lens, g, scale)
    row_bound, state_bound = bounds(q, k, v, lens, g, scale)
    T = sum(lens)
    check(out[:T], want[:T], row_bound[:T], dtype)
    check(state[slots.to(DEV)], ends, state_bound)
    assert (out[T:] == 7).all()
    rest = torch.ones(len(state), dtype=torch.bool)
    rest[slots] = False
    assert (state[rest.to(DEV)] == 9).all()


@pytest.mark.parametrize("kind", ["windows", "edges"])
@pytest.mark.parametrize("dtype,H,KV,D", [(torch.bfloat16, 8, 2, 128), (torch.float16, 5, 5, 64), (torch.bfloat16, 5, 1, 256)])
@pytest.mark.parametrize("lens", [(0, 1, 70), (130, 600, 3)])
def test_prompts_from_states_in_place_and_across_slots(lens, dtype, H, KV, D, kind):
    q, k, v, cu = inputs(lens, H, KV, D, dtype, seed=2, fused=True)
    g, scale = decays(H, kind), -0.3
    pool = torch.randn(8, H, D, D, generator=torch.Generator().manual_seed(3)).to(DEV) * 4
    read, write = ints([5, 2, -1]), ints([5, 7, -4])  # in place, to another slot, from zeros and not kept
    starts = torch.stack([pool[5], pool[2], torch.zeros_like(pool[0])])
    state, out = pool.clone(), torch.empty(len(q), H, D, device=DEV)
    linear_prompt(q, k, v, cu, g, scale, out, state, read, write)
    want, ends = linear64(q, k, v, lens, g, scale, starts)
    row_bound, state_bound = bounds(q, k, v, lens, g, scale, starts)
    check(out, want, row_bound)
    check(state[5], ends[0], state_bound[0])
    check(state[7], ends[1], state_bound[1])
    for slot in (0, 1, 2, 3, 4, 6):
        assert torch.equal(state[slot], pool[slot])


def test_a_prompt_in_pieces_ends_where_the_whole_one_does():
    lens, H, KV, D = (700,), 4, 2, 128
    q, k, v, cu = inputs(lens, H, KV, D, torch.bfloat16, seed=4)
    g, scale = decays(H), D ** -0.5
    want, ends = linear64(q, k, v, lens, g, scale)
    row_bound, state_bound = bounds(q, k, v, lens, g, scale)
    state, out, at = torch.zeros(1, H, D, D, device=DEV), torch.empty(700, H, D, device=DEV), 0
    for n in (1, 64, 37, 513, 85):
        part = slice(at, at + n)
        if n == 1:
            linear_step(q[part], k[part], v[part], g, scale, out[part], state, ints([0]), ints([0]))
        else:
            linear_prompt(q[part], k[part], v[part], ints([0, n]), g, scale, out[part], state, ints([0]), ints([0]))
        at += n
    check(out, want, 2 * row_bound)  # each piece rounds its state to fp32 once, as the whole does between parts
    check(state, ends, 2 * state_bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,H,KV,D", [(1, 1, 1, 64), (3, 8, 2, 128), (70, 4, 4, 64), (5, 2, 1, 256)])
@pytest.mark.parametrize("out_dtype", [torch.float32, None])
def test_step(n, H, KV, D, dtype, out_dtype):
    q, k, v, _ = inputs((n,), H, KV, D, dtype, seed=5, fused=True)
    g, scale = decays(H), D ** -0.5
    pool = torch.randn(2 * n + 1, H, D, D, generator=torch.Generator().manual_seed(6)).to(DEV) * 4
    gen = torch.Generator().manual_seed(7)
    read = torch.randint(0, n, (n,), generator=gen)  # some slots are read twice
    write = torch.randperm(n, generator=gen) + n
    state, out = pool.clone(), torch.empty(n, H, D, device=DEV, dtype=out_dtype or dtype)
    assert linear_step(q, k, v, g, scale, out, state, ints(read.tolist()), ints(write.tolist())) is out
    starts, lens = pool[read.to(DEV)], (1,) * n
    want, ends = linear64(q, k, v, lens, g, scale, starts)
    row_bound, state_bound = bounds(q, k, v, lens, g, scale, starts)
    check(out, want, row_bound, out.dtype)
    check(state[write.to(DEV)], ends, state_bound)
    assert torch.equal(state[:n], pool[:n]) and torch.equal(state[2 * n:], pool[2 * n:])
    # in place: the same bits
    again, other = pool.clone(), torch.empty_like(out)
    again[:n] = pool[read.to(DEV)]
    own = ints(range(n))
    linear_step(q, k, v, g, scale, other, again, own, own)
    assert torch.equal(other, out) and torch.equal(again[:n], state[write.to(DEV)])


def test_step_from_nothing_and_to_nowhere():
    q, k, v, _ = inputs((3,), 2, 1, 64, torch.bfloat16, seed=8)
    g = decays(2)
    state = torch.ones(2, 2, 64, 64, device=DEV)
    out = torch.empty(3, 2, 64, device=DEV)
    linear_step(q, k, v, g, 0.5, out, state, None, None)
    want, _ = linear64(q, k, v, (1, 1, 1), g, 0.5)
    check(out, want, bounds(q, k, v, (1, 1, 1), g, 0.5)[0])
    assert (state == 1).all()
    other = torch.empty_like(out)
    linear_step(q, k, v, g, 0.5, other, state, ints([-1, -7, -1]), ints([-1, -1, -2]))
    assert torch.equal(out, other) and (state == 1).all()


@pytest.mark.parametrize("lens", [(5, 600, 40, 3), (1, 1, 1, 1)])
@pytest.mark.parametrize("read,write,bad", [
    ([0, 1, 2, 3], [4, 4, 6, 7], {0, 1}),       # two write one slot
    ([0, 1, 2, 3], [4, 5, 0, 7], {0, 2}),       # one writes what another reads
    ([0, 1, 2, 8], [4, 5, 6, 7], {3}),          # a slot that is not there
    ([0, 1, 2, 3], [4, 5, 6, 1 << 30], {3}),
    ([0, 0, 0, 0], [4, 5, 6, 7], set()),        # all read one slot
])
def test_slots_that_meet_are_refused_by_their_sequences(lens, read, write, bad):
    H, D = 2, 64
    q, k, v, cu = inputs(lens, H, H, D, torch.bfloat16, seed=9)
    g = decays(H)
    pool = torch.randn(8, H, D, D, generator=torch.Generator().manual_seed(10)).to(DEV)
    for step in ((False, True) if max(lens) == 1 else (False,)):
        state, out = pool.clone(), torch.empty(len(q), H, D, device=DEV)
        if step:
            linear_step(q, k, v, g, 1.0, out, state, ints(read), ints(write))
        else:
            linear_prompt(q, k, v, cu, g, 1.0, out, state, ints(read), ints(write))
        at = 0
        for i, n in enumerate(lens):
            rows = out[at:at + n]
            at += n
            if i in bad:
                assert torch.isnan(rows).all()
                if 0 <= write[i] < 8:
                    assert torch.equal(state[write[i]], pool[write[i]])
            else:
                assert torch.isfinite(rows).all() and not torch.equal(state[write[i]], pool[write[i]])


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 256)])
@pytest.mark.parametrize("what", ["q", "k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_infinities_and_nan_reach_later_rows_only(dtype, D, what, value):
    lens, H = (200, 90, 600), 2
    q, k, v, cu = inputs(lens, H, 1, D, dtype, seed=11)
    g, scale = torch.full((H,), -0.01, device=DEV), D ** -0.5
    run = lambda: (linear_prompt(q, k, v, cu, g, scale, torch.empty(len(q), H, D, device=DEV, dtype=dtype), state, None, ints([0, 1, 2])), state.clone())
    state = torch.zeros(3, H, D, D, device=DEV)
    before, ends = run()
    for row in (200 + 37, 290 + 530):
        {"q": q, "k": k, "v": v}[what][row, 0, 5] = value
    after, ends2 = run()
    bits = lambda x: x.contiguous().view(torch.int16)
    assert torch.equal(bits(after[:237]), bits(before[:237])) and torch.equal(bits(after[290:820]), bits(before[290:820]))
    assert torch.equal(ends2[0], ends[0])
    if what == "q":  # that row of that head alone
        hit = torch.zeros_like(after, dtype=torch.bool)
        hit[237, 0] = hit[820, 0] = True
        assert not torch.isfinite(after[hit]).any() and torch.equal(bits(after)[~hit], bits(before)[~hit]) and torch.equal(ends, ends2)
        return
    for lo, hi, end in ((237, 290, ends2[1]), (820, 890, ends2[2])):
        if what == "v":  # that dim of every head, and the state's column
            assert not torch.isfinite(after[lo:hi, :, 5]).any() and not torch.isfinite(end[:, :, 5]).any()
            rest = torch.arange(D) != 5
            assert torch.isfinite(after[lo:hi][..., rest.to(DEV)]).all() and torch.isfinite(end[..., rest.to(DEV)]).all()
        else:  # every dim
            assert not torch.isfinite(after[lo:hi]).any() and not torch.isfinite(end[:, 5]).any()


@pytest.mark.parametrize("H,KV,D", [(8, 2, 128), (2, 2, 64), (2, 1, 256)])
def test_bits_do_not_depend_on_the_batch(H, KV, D):
    lens = (3, 700, 64, 1, 513)
    q, k, v, cu = inputs(lens, H, KV, D, torch.bfloat16, seed=12)
    g = decays(H)
    pool = torch.randn(10, H, D, D, generator=torch.Generator().manual_seed(13)).to(DEV)
    state, out = pool.clone(), torch.empty(len(q), H, D, device=DEV)
    linear_prompt(q, k, v, cu, g, 0.1, out, state, ints(range(5)), ints(range(5, 10)))
    at = 0
    for i, n in enumerate(lens):
        part = slice(at, at + n)
        alone, o = pool[i:i + 1].clone(), torch.empty(n, H, D, device=DEV)
        linear_prompt(q[part], k[part], v[part], ints([0, n]), g, 0.1, o, alone, ints([0]), ints([0]))
        assert torch.equal(o, out[part]) and torch.equal(alone[0], state[5 + i])
        at += n


@pytest.mark.parametrize("dtype,magnitude", [(torch.float16, 300.0), (torch.float16, 1e-4), (torch.bfloat16, 1e10), (torch.bfloat16, 1e-9)])
def test_magnitudes(dtype, magnitude):
    lens, H, D = (150,), 2, 64
    q, k, v, cu = inputs(lens, H, H, D, dtype, seed=14, magnitude=magnitude)
    g = decays(H)
    out, state = torch.empty(150, H, D, device=DEV), torch.empty(1, H, D, D, device=DEV)
    linear_prompt(q, k, v, cu, g, 1.0, out, state, None, ints([0]))
    want, ends = linear64(q, k, v, lens, g, 1.0)
    row_bound, state_bound = bounds(q, k, v, lens, g, 1.0)
    check(out, want, row_bound)
    check(state, ends, state_bound)


@pytest.mark.parametrize("step", [False, True])
def test_captured_on_another_stream(step):
    lens = (1,) * 6 if step else (530, 3, 65)
    H, D = 2, 128
    q, k, v, cu = inputs(lens, H, 1, D, torch.bfloat16, seed=15)
    g, n = decays(H), len(lens)
    pool = torch.randn(2 * n, H, D, D, generator=torch.Generator().manual_seed(16)).to(DEV)
    state, out = pool.clone(), torch.empty(len(q), H, D, device=DEV)
    read, write = ints(range(n)), ints(range(n, 2 * n))

    def call(out, state):
        if step:
            linear_step(q, k, v, g, 1.0, out, state, read, write)
        else:
            linear_prompt(q, k, v, cu, g, 1.0, out, state, read, write)

    call(out, state)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    other, there = torch.empty_like(out), pool.clone()
    with torch.cuda.stream(side):
        call(other, there)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(other, there)
    for i in range(3):
        other.zero_()
        there.copy_(pool)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(other, out) and torch.equal(there, state)
        call(torch.empty_like(out), pool.clone())


def test_strided_states_and_the_statement():
    lens, H, D = (70, 2), 2, 64
    q, k, v, cu = inputs(lens, H, 1, D, torch.bfloat16, seed=17)
    g = decays(H)
    wide = torch.zeros(4, 3 * H, D, D, device=DEV)  # every third head, of every other slot
    state = wide[::2, 1::3]
    out = torch.empty(72, H, D, device=DEV)
    linear_prompt(q, k, v, cu, g, 0.5, out, state, None, ints([1, 0]))
    row_bound, state_bound = bounds(q, k, v, lens, g, 0.5)
    said = torch.zeros(2, H, D, D, device=DEV)
    check(out, linear_attention_torch(q, k, v, cu, g, 0.5, said, None, ints([1, 0])).double(), 2 * row_bound)
    check(state[[1, 0]], said[[1, 0]].double(), 2 * state_bound)
    assert not wide[1::2].any() and not wide[::2, ::3].any() and not wide[::2, 2::3].any()


def test_empty_calls():
    e = torch.empty(0, 2, 64, device=DEV, dtype=torch.bfloat16)
    g = decays(2)
    state = torch.ones(2, 2, 64, 64, device=DEV)
    linear_step(e, e, e, g, 1.0, e.clone(), state, ints([]), ints([]))
    linear_prompt(e, e, e, ints([0]), g, 1.0, e.clone())
    linear_prompt(e, e, e, ints([0, 0]), g, 1.0, e.clone(), state, ints([-1]), ints([0]))  # zeros are where it starts and ends
    assert not state[0].any() and (state[1] == 1).all()


def test_refusals():
    q, k, v, cu = inputs((4,), 2, 1, 64, torch.bfloat16)
    g, out, state = decays(2), torch.empty(4, 2, 64, device=DEV), torch.zeros(2, 2, 64, 64, device=DEV)
    slots = ints([0])
    ok = dict(q=q, k=k, v=v, cu=cu, g=g, scale=1.0, out=out, state=state, read=None, write=slots)
    for over, kind in ((dict(q=q.float()), NotImplementedError), (dict(k=k.half()), NotImplementedError), (dict(out=out.double()), ValueError),
                       (dict(cu=cu.long()), ValueError), (dict(g=g.double()), ValueError), (dict(g=g[:1]), ValueError),
                       (dict(state=state.bfloat16()), NotImplementedError), (dict(state=state[:, :1]), ValueError), (dict(state=None), ValueError),
                       (dict(state=state.transpose(2, 3)), ValueError), (dict(write=slots.long()), ValueError), (dict(write=ints([0, 1])), ValueError),
                       (dict(k=k[:3]), ValueError), (dict(q=q[..., :32], k=k[..., :32], v=v[..., :32], out=out[..., :32], state=None, write=None), NotImplementedError),
                       (dict(scale="x"), TypeError), (dict(write="x"), TypeError)):
        with pytest.raises(kind):
            linear_prompt(*dict(ok, **over).values())


def test_many_sequences_and_starts_beyond_the_rows():
    """More sequences than a wave has lanes, empty ones among them, long ones at both ends: each as it is alone."""
    g = torch.Generator().manual_seed(18)
    lens = [600, 0] + torch.randint(0, 40, (195,), generator=g).tolist() + [512, 0, 1025]
    H, D = 2, 64
    q, k, v, cu = inputs(lens, H, 1, D, torch.bfloat16, seed=19)
    gd, n = decays(H), len(lens)
    state, out = torch.zeros(n, H, D, D, device=DEV), torch.empty(len(q), H, D, device=DEV)
    linear_prompt(q, k, v, cu, gd, 0.125, out, state, None, ints(range(n)))
    for i in [0, 1, 2, 63, 64, 65, 130, n - 3, n - 2, n - 1]:
        lo, hi = int(cu[i]), int(cu[i + 1])
        alone, o = torch.ones(1, H, D, D, device=DEV), torch.empty(hi - lo, H, D, device=DEV)
        linear_prompt(q[lo:hi], k[lo:hi], v[lo:hi], ints([0, hi - lo]), gd, 0.125, o, alone, None, ints([0]))
        assert torch.equal(o, out[lo:hi]) and torch.equal(alone[0], state[i]), i
    # a last start beyond the rows ends at them; starts that fall back make sequences of no rows
    rows = len(q)
    other = torch.full_like(out, 5.0)
    linear_prompt(q, k, v, ints([-3, 700, rows + 1000]), gd, 0.125, other)
    again = torch.full_like(out, 5.0)
    linear_prompt(q, k, v, ints([0, 700, rows]), gd, 0.125, again)
    assert torch.equal(other, again)
    linear_prompt(q, k, v, ints([10, 20, 5, 5]), gd, 0.125, other.fill_(5.0))
    assert (other[:10] == 5).all() and (other[20:] == 5).all() and torch.isfinite(other).all()


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_of_the_output_anywhere(out_dtype):
    lens, H, D = (40, 70), 2, 128
    q, k, v, cu = inputs(lens, H, 1, D, torch.bfloat16, seed=20)
    g, state = decays(H), torch.zeros(2, H, D, D, device=DEV)
    wide = torch.full((110, 3, D + 3), 2.0, device=DEV, dtype=out_dtype)
    out = wide[:, :H, 1:D + 1]  # rows at odd elements
    linear_prompt(q, k, v, cu, g, 0.25, out, state, None, ints([0, 1]))
    want, _ = linear64(q, k, v, lens, g, 0.25)
    row_bound, _ = bounds(q, k, v, lens, g, 0.25)
    check(out, want, row_bound, out_dtype)
    assert (wide[:, H:] == 2).all() and (wide[..., 0] == 2).all() and (wide[..., D + 1:] == 2).all()
    n = len(q)
    linear_step(q, k, v, g, 0.25, out, torch.zeros(1, H, D, D, device=DEV), None, None)
    want, _ = linear64(q, k, v, (1,) * n, g, 0.25)
    check(out, want, bounds(q, k, v, (1,) * n, g, 0.25)[0], out_dtype)


def test_a_step_in_many_steps_keeps_its_bits_of_the_decay():
    """4000 tokens with a window of 10000: the decay's own rounding (2^-25) would add up to 4000 of it."""
    H, D, n = 1, 64, 4000
    g = torch.full((H,), -1e-4, device=DEV)
    state = torch.ones(1, H, D, D, device=DEV)
    zero, out = torch.zeros(1, H, D, device=DEV, dtype=torch.bfloat16), torch.empty(1, H, D, device=DEV)
    for _ in range(n):
        linear_step(zero, zero, zero, g, 1.0, out, state, ints([0]), ints([0]))
    want = torch.exp(g.double() * n)
    # one rounding of 2^-24 a step, to the nearest: a walk of sqrt(4000) of half steps, with room for six of its deviations
    assert (state.double() / want - 1).abs().max() < 6 * n ** 0.5 * 2.0 ** -24


@pytest.mark.parametrize("step", [False, True])
def test_rows_and_states_far_apart(step):
    """Rows of the longest stride there is, past 2^31 elements and 2^32 bytes; two states as far from each other."""
    n, H, D, stride = 300, 2, 64, (1 << 23) - 8
    q, k, v, cu = inputs((n,), H, 1, D, torch.bfloat16, seed=21)
    g = decays(H)

    def far(x):
        y = torch.empty(stride * (n - 1) + x.shape[1] * D, device=DEV, dtype=x.dtype).as_strided(x.shape, (stride, D, 1))
        return y.copy_(x)

    fq, fk, fv, out = far(q), far(k), far(v), far(q)
    pool = torch.empty((1 << 31) + 16 + H * D * D, device=DEV).as_strided((2, H, D, D), ((1 << 31) + 16, D * D, D, 1))
    starts = torch.randn(n if step else 1, H, D, D, generator=torch.Generator().manual_seed(22)).to(DEV)
    lens = (1,) * n if step else (n,)
    if step:
        pool[0], pool[1] = starts[0], 3.0
        starts[:] = starts[0].clone()
        read, write = ints([0] * n), ints([-1] * (n - 1) + [1])
        linear_step(fq, fk, fv, g, 0.5, out, pool, read, write)
    else:
        pool[0], pool[1] = 3.0, starts[0]
        linear_prompt(fq, fk, fv, cu, g, 0.5, out, pool, ints([1]), ints([1]))
    want, ends = linear64(q, k, v, lens, g, 0.5, starts)
    row_bound, state_bound = bounds(q, k, v, lens, g, 0.5, starts)
    check(out, want, row_bound, torch.bfloat16)
    check(pool[1], ends[-1], state_bound[-1])
    assert torch.equal(pool[0], starts[0]) if step else (pool[0] == 3).all()


def test_two_calls_at_once():
    calls = []
    for seed in (23, 24):
        q, k, v, cu = inputs((3000, 40, 700), 4, 2, 128, torch.bfloat16, seed=seed)
        calls.append((q, k, v, cu, decays(4), 0.1))
    want = []
    for c in calls:
        state = torch.zeros(3, 4, 128, 128, device=DEV)
        want.append((linear_prompt(*c, torch.empty_like(c[0]), state, None, ints([0, 1, 2])), state))
    got = [(torch.empty_like(c[0]), torch.zeros(3, 4, 128, 128, device=DEV), ints([0, 1, 2])) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, (out, state, slots), stream in zip(calls, got, streams):
            with torch.cuda.stream(stream):
                linear_prompt(*c, out, state, None, slots)
    torch.cuda.synchronize()
    for (out, state, _), (a, b) in zip(got, want):
        assert torch.equal(out, a) and torch.equal(state, b)


def test_outputs_over_the_inputs_are_refused():
    q, k, v, cu = inputs((5,), 2, 2, 64, torch.bfloat16)
    pool, slots = torch.zeros(5, 2, 64, 64, device=DEV), torch.arange(5, dtype=torch.int32, device=DEV)
    for out in (q, k, v):
        with pytest.raises(ValueError, match="out must not be"):
            linear_prompt(q, k, v, cu, decays(2), 0.1, out)
        with pytest.raises(ValueError, match="out must not be"):
            linear_step(q, k, v, decays(2), 0.1, out, pool, slots, slots)


@pytest.mark.parametrize("dtype,H,KV,D", [(torch.bfloat16, 16, 4, 64), (torch.bfloat16, 17, 17, 64), (torch.float16, 20, 5, 128), (torch.float16, 18, 2, 256), (torch.bfloat16, 6, 3, 256)])
@pytest.mark.parametrize("lens", [(319, 320, 321), (511, 512, 513, 0, 3), (961, 1, 640), (383, 385, 769), (1536, 1537)])
def test_lengths_about_the_parts(lens, dtype, H, KV, D):
    """Sequences are cut into parts whose length goes by the heads: lengths beside their multiples, from states, in place."""
    q, k, v, cu = inputs(lens, H, KV, D, dtype, seed=26, extra=1)
    g, scale = decays(H), D ** -0.5
    starts = torch.randn(len(lens), H, D, D, generator=torch.Generator().manual_seed(27)).to(DEV)
    state, slots = starts.clone(), torch.arange(len(lens), dtype=torch.int32, device=DEV)
    out = torch.full((len(q), H, D), 7.0, device=DEV)
    linear_prompt(q, k, v, cu, g, scale, out, state, slots, slots)
    want, ends = linear64(q, k, v, lens, g, scale, starts)
    row_bound, state_bound = bounds(q, k, v, lens, g, scale, starts)
    check(out[:-1], want[:-1], row_bound[:-1])
    check(state, ends, state_bound)
    assert (out[-1] == 7).all()
